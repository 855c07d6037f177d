// Key bounds of cache blocks, and the blocks that promise a query row the most.
//
// Bounds: of each block and kv head the int8 codes of every dim's least and largest
// key value, rounded outwards, times one power of two: the least 2^e, e >= -100, at
// which the largest magnitude is at most 127.  Past 127 x 2^100, and for infinities
// and NaN, the block is open (exponent byte 255): it bounds nothing.  A record is
// [Hkv][lo D bytes | hi D bytes], then Hkv exponent bytes (e + 128), padded to 16.
//
// Scores: the G heads of a (row, kv head) are rounded to int8 codes c by the same
// rule with one power of two, and a block's score is 2^e max_g sum_d max(c lo, c hi),
// open blocks +infinity.  max(c lo, c hi) = max(c, 0) hi + min(c, 0) lo, so the sum is an int8
// dot product of length 2 D on v_mfma_i32_16x16x64_i8.  It is a whole number below
// 2^24 (2 D x 127^2 at most 8.3 million), so the fp32 score is exact and the selection
// is the same whatever the order of the sums; ties go to the lower block.  Up to c's
// rounding no key of the block scores higher.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "generic.h"
#include "launch.h"

namespace gllm {

typedef __attribute__((ext_vector_type(4))) int i32x4;

// 127 x 2^100 as fp32 bits
constexpr uint32_t kCodeMax = ((100u + 6 + 127) << 23) | 0x7e0000u;
constexpr int kOpen = 255;
// Least e >= -100 with x <= 127 x 2^e = 1.984375 x 2^(e + 6), x's bits at most kCodeMax.
__device__ __forceinline__ int code_exponent(uint32_t bits) {
  const int e = (int)(bits >> 23) - 127 - 6 + ((bits & 0x7fffffu) > 0x7e0000u);
  return max(e, -100);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// 8 values of a row of the model dtype
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    float v[8];
    __builtin_memcpy(v, p, 32);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[i];
  } else {
    u32x4 w;
    __builtin_memcpy(&w, p, 16);
    unpack8<T>(w, x);
  }
}
// 8 cached values as attention reads them: in the model dtype QT
template <typename KV, typename QT>
__device__ __forceinline__ void load8_kv(const void* row, int d, const uint8_t* scales, float* x) {
  if constexpr (std::is_same<KV, kv4>::value) {
    uint32_t w;
    __builtin_memcpy(&w, (const uint8_t*)row + d / 2, 4);
    const float scale = __uint_as_float((uint32_t)scales[d / 32] << 23);
#define GLLM_PAIR(i)                                                          \
  {                                                                           \
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, i);     \
    x[2 * i] = v[0];                                                          \
    x[2 * i + 1] = v[1];                                                      \
  }
    GLLM_PAIR(0) GLLM_PAIR(1) GLLM_PAIR(2) GLLM_PAIR(3)
#undef GLLM_PAIR
  } else if constexpr (std::is_same<KV, fp8e4m3>::value) {
    u32x2 w;
    __builtin_memcpy(&w, (const uint8_t*)row + d, 8);
    unpack_fp8x4(w[0], x);
    unpack_fp8x4(w[1], x + 4);
  } else {
    load8<KV>((const KV*)row + d, x);
  }
  constexpr bool exact = std::is_same<QT, float>::value || std::is_same<KV, QT>::value || std::is_same<KV, fp8e4m3>::value;
  if constexpr (!exact) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = rnd<QT>(x[i]);
  }
}

// ---------------------------------------------------------------- key bounds
// One workgroup per (block, kv heads of at most kBoundsDims dims): a thread takes 8 dims of
// a head over every KG-th key, the KG parts and the heads' magnitudes meet in LDS.
// Reads the block's keys once; HBM-bound for prompts, one latency for a decode step.
constexpr int kBoundsThreads = 256;
constexpr int kBoundsDims = 2048;
template <typename KV, typename QT>
__global__ void __launch_bounds__(kBoundsThreads) key_bounds_kernel(BoundsArgs a, int heads) {
  // [part][lo, hi][dims]: one part where a thread per 8 dims takes them all
  __shared__ __attribute__((aligned(16))) float part[2 * kBoundsDims];
  __shared__ uint32_t top[kBoundsDims / 8];
  const int D = a.head_dim, h0 = blockIdx.y * heads, nh = min(heads, a.num_kv_heads - h0);
  const BoundsBlock bb = a.blocks[blockIdx.x];
  const int tid = threadIdx.x, nc = nh * D / 8;          // 8-dim chunks, at most 256
  uint32_t blk = (uint32_t)a.block_table[(int64_t)bb.seq * a.block_table_stride + bb.block];
  if (blk >= (uint64_t)a.num_blocks) return;             // outside the pool: no record
  for (int i = tid; i < nh; i += kBoundsThreads) top[i] = 0u;
  // parts of the keys: as many as threads and LDS hold
  const int kg = max(1, min(kBoundsThreads / nc, kBoundsDims / (nh * D)));
  const int g = tid / nc, c = tid - g * nc;
  float lo[8], hi[8];
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] = -kNegInf;
    hi[i] = kNegInf;
  }
  const int hh = c * 8 / D, d = c * 8 - hh * D;          // head of the workgroup, first dim
  const auto load_key = [&](int t, float* x) {
    if constexpr (std::is_same<KV, kv4>::value) {
      const uint8_t* rec = (const uint8_t*)a.k_cache + (int64_t)blk * a.cache_slot_stride + (int64_t)(h0 + hh) * a.kv4_record;
      load8_kv<KV, QT>(rec + t * (D / 2), d, rec + (int64_t)a.block_size * (D / 2) + t * (D / 32), x);
    } else {
      const KV* row = (const KV*)a.k_cache + ((int64_t)blk * a.block_size + t) * a.cache_slot_stride + (int64_t)(h0 + hh) * D;
      load8_kv<KV, QT>(row, d, nullptr, x);
    }
  };
  __syncthreads();
  if (g < kg) {
    // four keys' loads at a time; past the last one it is read again
    for (int t0 = g; t0 < bb.n; t0 += 4 * kg) {
      float x[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) load_key(min(t0 + u * kg, bb.n - 1), x[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          lo[i] = fminf(lo[i], x[u][i]);
          hi[i] = fmaxf(hi[i], x[u][i]);
          m = max(m, magnitude(x[u][i]));                // a NaN's bits are above infinity's
        }
    }
    atomicMax(&top[hh], m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[(2 * g) * nc * 8 + c * 8 + i] = lo[i];
      part[(2 * g + 1) * nc * 8 + c * 8 + i] = hi[i];
    }
  }
  __syncthreads();
  uint8_t* rec = a.bounds + (int64_t)blk * a.bounds_stride;
  if (tid < nh) rec[(int64_t)a.num_kv_heads * 2 * D + h0 + tid] = top[tid] > kCodeMax ? kOpen : code_exponent(top[tid]) + 128;
  if (g > 0 || c >= nc) return;
  for (int k = 1; k < kg; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = fminf(lo[i], part[(2 * k) * nc * 8 + c * 8 + i]);
      hi[i] = fmaxf(hi[i], part[(2 * k + 1) * nc * 8 + c * 8 + i]);
    }
  const bool open = top[hh] > kCodeMax;
  const float inv = open ? 0.f : pow2f(-code_exponent(top[hh]));
  uint32_t wl[2] = {0u, 0u}, wh[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // exact but for an underflow to 0, which still has its sign
    int cl = (int)floorf(lo[i] * inv), ch = (int)ceilf(hi[i] * inv);
    if (lo[i] < 0.f && cl == 0) cl = -1;
    if (hi[i] > 0.f && ch == 0) ch = 1;
    if (open) cl = ch = 0;
    wl[i / 4] |= (uint32_t)(uint8_t)(int8_t)cl << (8 * (i % 4));
    wh[i / 4] |= (uint32_t)(uint8_t)(int8_t)ch << (8 * (i % 4));
  }
  uint8_t* dst = rec + (int64_t)(h0 + hh) * 2 * D + d;
  st8(dst, u32x2{wl[0], wl[1]});
  st8(dst + D, u32x2{wh[0], wh[1]});
}

template <typename QT>
static hipError_t launch_bounds_t(const BoundsArgs& a, dim3 grid, int heads, hipStream_t st) {
  const dim3 block(kBoundsThreads);
  switch (a.kv_dtype) {
    case kF32: hipLaunchKernelGGL((key_bounds_kernel<float, QT>), grid, block, 0, st, a, heads); break;
    case kBF16: hipLaunchKernelGGL((key_bounds_kernel<__bf16, QT>), grid, block, 0, st, a, heads); break;
    case kF16: hipLaunchKernelGGL((key_bounds_kernel<_Float16, QT>), grid, block, 0, st, a, heads); break;
    case kFP8: hipLaunchKernelGGL((key_bounds_kernel<fp8e4m3, QT>), grid, block, 0, st, a, heads); break;
    case kMXFP4: hipLaunchKernelGGL((key_bounds_kernel<kv4, QT>), grid, block, 0, st, a, heads); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}
hipError_t launch_key_bounds(const BoundsArgs& a, hipStream_t st) {
  if (a.n_blocks == 0) return hipSuccess;
  const int heads = kBoundsDims / a.head_dim;
  const dim3 grid(a.n_blocks, (a.num_kv_heads + heads - 1) / heads);
  switch (a.dtype) {
    case kF32: return launch_bounds_t<float>(a, grid, heads, st);
    case kBF16: return launch_bounds_t<__bf16>(a, grid, heads, st);
    case kF16: return launch_bounds_t<_Float16>(a, grid, heads, st);
    default: return hipErrorInvalidValue;
  }
}

// A thread per 4 codes.
__global__ void __launch_bounds__(256) key_bounds_values_kernel(BoundsValuesArgs a, int64_t total) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= total) return;
  const int D = a.head_dim, per = a.num_kv_heads * 2 * D / 4;
  const int64_t b = e / per;
  const int at = (int)(e - b * per) * 4, h = at / (2 * D);
  const int64_t blk = a.blocks[b];
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (blk >= 0 && blk < a.num_blocks) {
    const uint8_t* rec = a.bounds + blk * a.bounds_stride;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + at);
    const int byte = rec[a.num_kv_heads * 2 * D + h];
    // any byte, also one that no writer leaves: 2^(byte - 128) from 2^-128 on
    const float scale = byte == 0 ? __uint_as_float(0x00200000u) : byte == 1 ? __uint_as_float(0x00400000u) : pow2f(byte - 128);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i)) * scale;
    if (byte == kOpen) x = at - h * 2 * D < D ? f32x4{kNegInf, kNegInf, kNegInf, kNegInf} : f32x4{-kNegInf, -kNegInf, -kNegInf, -kNegInf};
  }
  *reinterpret_cast<f32x4*>(a.out + 4 * e) = x;
}
hipError_t launch_key_bounds_values(const BoundsValuesArgs& a, hipStream_t st) {
  const int64_t total = a.n_blocks * (a.num_kv_heads * 2 * a.head_dim / 4);
  if (total == 0) return hipSuccess;
  if ((total + 255) / 256 > INT32_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL(key_bounds_values_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, a, total);
  return hipGetLastError();
}

// ---------------------------------------------------------------- scores
// One 8-wave workgroup per (item: a tile of query rows and a run of 16-block groups; HW
// kv heads); a wave takes one of the heads and its share of the groups, two groups'
// loads ahead.  A column of the MFMA is a (row of the tile, head of the group) pair, n = row x
// GP + g with GP = G rounded up to a power of two (columns past G repeat the last head), so
// a tile's rows share the bounds they load; more than 16 heads go by in passes.  Lane (n, grp)
// loads bytes 64 s + 16 grp .. + 15 of block n's [lo | hi]; the codes of q lie in the same
// order.  Blocks are the product's columns, so a lane has one block's scale and up to four
// heads of a row to reduce.
// Decode rows are HBM-bound (64 rows on 8,192-32,768 keys, blocks of 16: 170 MB in 33 us
// from cache, ~44 from HBM).  Prompt rows are bound by the CU's loads, which take the 16
// records of an instruction one by one: 840 rows on 8,192-16,384 keys, blocks of 32, make
// 37,300 cache accesses on each of 212 CUs in some 40,000 cycles.  RT = 2 tiles of 16 columns
// on the same loads, one workgroup a CU for its registers, cut them from 28.2 to 19.9 us (four:
// 20.2).
constexpr int kScoreWaves = 8;
// The maximum over lanes {l, l ^ 16} and {l, l ^ 32}.
__device__ __forceinline__ int columns_max16(int v) {
  const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  return max((int)r[0], (int)r[1]);
}
__device__ __forceinline__ int columns_max32(int v) {
  const auto r = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return max((int)r[0], (int)r[1]);
}
constexpr int kScorePF = 2;
template <typename QT, int NK, int GP, int RT, bool PASSES>
__global__ void __launch_bounds__(64 * kScoreWaves) __attribute__((amdgpu_waves_per_eu(NK == 8 || RT > 1 || PASSES ? 2 : 4))) block_scores_kernel(SelectArgs a, int hw) {
  const int lane = threadIdx.x & 63, n = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int D = a.head_dim, G = a.num_q_heads / a.num_kv_heads, Hkv = a.num_kv_heads;
  const int hgs = Hkv / hw;
  const ScoreItem tl = a.items[a.item0 + blockIdx.x / hgs];
  const int h = blockIdx.x % hgs * hw + wave % hw;
  const int kw = kScoreWaves / hw;                       // waves of a head, their groups one after another
  const int share = (tl.groups + kw - 1) / kw, first = wave / hw * share;
  const int b0 = (tl.group0 + first) * 16;
  const int ng = min(share, tl.groups - first);
  if (ng <= 0) return;
  static_assert(RT == 1 || !PASSES, "heads or rows fill the columns");
  constexpr int TR = 16 / GP;                            // rows of 16 columns
  const int g0 = n % GP, nt = RT == 1 ? 1 : (tl.nrows + TR - 1) / TR;
  static_assert(RT <= 2, "tile indexes are compile-time constants");
  const auto each_tile = [&](auto f) {
    f(std::integral_constant<int, 0>());
    if constexpr (RT > 1) f(std::integral_constant<int, 1>());
  };
  bool row_ok[RT];
  int row[RT];
  each_tile([&](auto t) {
    const int ri = t * TR + n / GP;
    row_ok[t] = ri < tl.nrows;
    row[t] = a.rows[tl.row0 + (row_ok[t] ? ri : 0)].row;
  });
  const int passes = PASSES ? (G + 15) / 16 : 1;
  // a byte of the word that is loaded (a byte load's value is widened where the loop ends,
  // which waits for every load in flight)
  struct Group { u32x4 box[NK]; uint32_t e; };
  const int32_t* bt = a.block_table + (int64_t)tl.seq * a.block_table_stride;
  // the pool's blocks of 16 groups, 64 a register, so that no load waits in the loop for
  // the older ones, which loads return in order
  constexpr int NI = 4;
  uint32_t ids[NI];
  const auto load_ids = [&](int u0) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint32_t blk = (uint32_t)bt[min(b0 + 16 * u0 + 64 * i + lane, tl.nblocks - 1)];   // past the last: the last
      ids[i] = blk < (uint64_t)a.num_blocks ? blk : 0u;  // never address outside the pool
    }
  };
  const auto issue = [&](int u, Group& x) {              // group u of the 16
    const int i = u >> 2;
    const uint32_t src = i == 0 ? ids[0] : i == 1 ? ids[1] : i == 2 ? ids[2] : ids[3];
    const uint32_t blk = (uint32_t)__shfl((int)src, 16 * (u & 3) + n, 64);
    const uint8_t* rec = a.bounds + (int64_t)blk * a.bounds_stride;
    const uint8_t* box = rec + h * 2 * D + 16 * grp;
#pragma unroll
    for (int s = 0; s < NK; ++s)
      x.box[s] = 64 * s + 64 <= 2 * D ? ld16(box + 64 * s) : ld16(rec + h * 2 * D + min(64 * s + 16 * grp, 2 * D - 16));
    x.e = *reinterpret_cast<const uint32_t*>(rec + Hkv * 2 * D + (h & ~3));
  };
  Group ring[kScorePF + 1];
  load_ids(0);

  // q's codes: one power of two for all heads of the group, then each half's sign.  A
  // lane's dims of the lo half are those of its hi half where 64 divides D.
  constexpr int NH = NK / 2;
  const bool folded = D == 32 * NK && D % 64 == 0;
  const auto q_at = [&](auto t, int p) {
    return (const QT*)a.q + (int64_t)row[t] * a.q_row_stride + (int64_t)(h * G + min(16 * p + g0, G - 1)) * D;
  };
  const auto dim_at = [&](int s) {                       // first dim of the lane's s-th 8 bytes
    const int k = 64 * (s / 2) + 16 * grp + 8 * (s % 2);
    return min(k < D ? k : k - D, D - 8);
  };
  float x[2 * NH][8];
  const auto load_half = [&](auto t, int p, int half) {
    const QT* qp = q_at(t, p);
#pragma unroll
    for (int s = 0; s < 2 * NH; ++s) load8<QT>(qp + dim_at(s + half * 2 * NH), x[s]);
  };
  load_half(std::integral_constant<int, 0>(), 0, 0);
  __builtin_amdgcn_sched_barrier(0);                     // q first: its codes are made while bounds are on their way
#pragma unroll
  for (int u = 0; u < kScorePF; ++u) issue(u, ring[u]);
  __builtin_amdgcn_sched_barrier(0);
  bool none[RT];
  float inv[RT];
  u32x4 qb[RT][NK];
  const auto codes = [&](auto t, int p) {
    const QT* qp = q_at(t, p);
#pragma unroll
    for (int s = 0; s < 2 * NK; ++s) {
      const int k = 64 * (s / 2) + 16 * grp + 8 * (s % 2);
      const bool lo = k < D;                             // lo takes the negative codes, hi the positive ones
      float v[8];
      if (folded && passes == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x[s % (2 * NH)][i];
      } else {
        load8<QT>(qp + dim_at(s), v);
      }
      uint32_t w[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = __builtin_rintf(v[i] * inv[t]), c1 = lo ? fminf(c, 0.f) : fmaxf(c, 0.f);
        w[i / 4] = __builtin_amdgcn_cvt_pk_u8_f32(c1 + 128.f, i % 4, w[i / 4]);
      }
      // code + 128 as a byte is the code's with the top bit turned
      qb[t][s / 2][2 * (s % 2)] = none[t] || k >= 2 * D ? 0u : w[0] ^ 0x80808080u;
      qb[t][s / 2][2 * (s % 2) + 1] = none[t] || k >= 2 * D ? 0u : w[1] ^ 0x80808080u;
    }
  };
  each_tile([&](auto t) {
    uint32_t m = 0u;
    for (int p = 0; p < passes; ++p) {
      for (int half = 0; half < (folded ? 1 : 2); ++half) {
        if (t + p + half > 0) load_half(t, p, half);
#pragma unroll
        for (int s = 0; s < 2 * NH; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) m = max(m, magnitude(x[s][i]));
      }
    }
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
#pragma unroll
    for (int s = 1; s < GP; s *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, s, 64));
    none[t] = !row_ok[t] || m > kCodeMax;
    inv[t] = m > kCodeMax ? 0.f : pow2f(-code_exponent(m));
    codes(t, 0);
  });
  // lane (n, grp) holds block n's sums with columns 4 grp .. + 3: NS rows of the tile from
  // sr on, whose heads are in the lane (GP > 4: in it and its neighbours of the same n)
  constexpr int NS = GP < 4 ? 4 / GP : 1;
  const int sr = 4 * grp / GP;
  float* const sp = a.scores + ((int64_t)(tl.row0 + sr - a.row0) * Hkv + h) * a.score_stride;
  const auto score = [&](int u, const Group& x) {
    const int e = (int)(x.e >> (8 * (h & 3)) & 255u);
    // bytes that no writer leaves are limited, so that the score stays a number
    const float scale = pow2f(min(max(e - 128, -100), 100));
    const int b = b0 + 16 * u + n;
    each_tile([&](auto t) {
      if (t > 0 && t >= nt) return;
      int best[4] = {INT32_MIN, INT32_MIN, INT32_MIN, INT32_MIN};
      for (int p = 0; p < passes; ++p) {
        if (PASSES) codes(t, p);
        i32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NK; ++s)
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, qb[t][s]), __builtin_bit_cast(i32x4, x.box[s]), acc, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) best[j] = PASSES ? max(best[j], acc[j]) : acc[j];   // columns past G repeat the last head
      }
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        int v = best[GP < 4 ? GP * i : 0];
#pragma unroll
        for (int j = 1; j < (GP < 4 ? GP : 4); ++j) v = max(v, best[(GP < 4 ? GP * i : 0) + j]);
        if (GP > 4) v = columns_max16(v);
        if (GP > 8) v = columns_max32(v);
        if (t * TR + sr + i < tl.nrows && (GP <= 4 || 4 * grp % GP == 0) && b < a.score_stride)
          sp[(int64_t)(t * TR + i) * Hkv * a.score_stride + b] = e == kOpen ? -kNegInf : (float)v * scale;
      }
    });
  };
  for (int c0 = 0; c0 < ng; c0 += 4 * NI) {
    const int nc = min(4 * NI, ng - c0);
    if (c0 > 0) {
      load_ids(c0);
#pragma unroll
      for (int u = 0; u < kScorePF; ++u) issue(u, ring[u]);
    }
    int u0 = 0;
    for (; u0 + kScorePF < nc; u0 += kScorePF + 1) {
#pragma unroll
      for (int u = 0; u <= kScorePF; ++u) {
        issue(min(u0 + u + kScorePF, 4 * NI - 1), ring[(u + kScorePF) % (kScorePF + 1)]);
        score(c0 + u0 + u, ring[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < kScorePF; ++u)
      if (u0 + u < nc) score(c0 + u0 + u, ring[u]);
  }
}

// ---------------------------------------------------------------- selection
// For each (row, kv head) the width-th largest key T by bisection over its bits, from
// the first one in which the candidates differ: a count of the keys above a candidate a
// step, until one keeps exactly as many.  Then the blocks above T and the first of those
// equal to it, in order.  Keys are the scores as unsigned integers of the same order;
// blocks that are always taken have the largest.
struct SelectRow {
  const float* scores;
  int32_t* out;
  int nb;
};
__device__ __forceinline__ SelectRow select_row(const SelectArgs& a, int unit) {
  const int ri = unit / a.num_kv_heads, h = unit - ri * a.num_kv_heads;
  const SparseRow sr = a.rows[a.row0 + ri];
  return {a.scores + ((int64_t)ri * a.num_kv_heads + h) * a.score_stride,
          a.selected + ((int64_t)sr.row * a.num_kv_heads + h) * a.width,
          (int)div_bs((uint32_t)sr.pos, a.block_magic, a.block_shift) + 1};
}
// The key of block b, whose score has the bits u: 0 behind the row, the largest if always taken.
__device__ __forceinline__ uint32_t score_key(const SelectArgs& a, const SelectRow& r, int b, uint32_t u) {
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return b >= r.nb ? 0u : b < a.first || b >= r.nb - a.recent ? 0xffffffffu : k;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) x = max(x, (uint32_t)__shfl_xor((int)x, s, 64));
  return x;
}

// One wave per (row, kv head), up to 64 NR blocks in its registers: no barriers, and
// the waves of a CU hide each other's steps.
constexpr int kWaveSelects = 4;
template <int NR>
__global__ void __launch_bounds__(64 * kWaveSelects) select_wave_kernel(SelectArgs a, int units) {
  const int lane = threadIdx.x & 63;
  const int unit = blockIdx.x * kWaveSelects + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (unit >= units) return;
  const SelectRow r = select_row(a, unit);
  const int K = a.width;
  if (r.nb <= K) {
    for (int j = lane; j < K; j += 64) r.out[j] = j < r.nb ? j : -1;
    return;
  }
  uint32_t keys[NR], hi = 0u, lo = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int b = lane + 64 * i;
    keys[i] = score_key(a, r, b, __float_as_uint(r.scores[min(b, r.nb - 1)]));
    const bool cand = b >= a.first && b < r.nb - a.recent;
    hi = max(hi, cand ? keys[i] : 0u);
    lo = min(lo, cand ? keys[i] : 0xffffffffu);
  }
  const auto count = [&](uint32_t c) {                    // keys >= c
    int n = 0;
#pragma unroll
    for (int i = 0; i < NR; ++i) n += __popcll(__builtin_amdgcn_ballot_w64(keys[i] >= c));
    return n;
  };
  uint32_t T = 0xffffffffu;
  int above = 0;                                          // keys > T
  if (K > a.first + a.recent) {                           // else only those always taken
    hi = __builtin_amdgcn_readfirstlane(wave_max(hi));
    lo = ~__builtin_amdgcn_readfirstlane(wave_max(~lo));
    int bit = hi == lo ? -1 : 31 - __clz((int)(hi ^ lo));
    T = bit < 0 ? hi : hi >> bit >> 1 << bit << 1;
    for (; bit >= 0; --bit) {
      const uint32_t c = T | (1u << bit);
      const int n = count(c);
      if (n >= K) T = c;
      if (n == K) break;                                  // exactly these
    }
    above = count(T + 1);                                 // T is no forced block's key
  }
  int eq_left = K - above, at = 0;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const uint64_t eq = __builtin_amdgcn_ballot_w64(keys[i] == T), gt = __builtin_amdgcn_ballot_w64(keys[i] > T);
    const uint64_t below = (1ull << lane) - 1;
    const int eq_mine = __popcll(eq & below);
    if (keys[i] > T || (keys[i] == T && eq_mine < eq_left))
      r.out[at + __popcll(gt & below) + min(eq_mine, eq_left)] = lane + 64 * i;
    const int taken = min(__popcll(eq), eq_left);
    at += __popcll(gt) + taken;
    eq_left -= taken;
  }
}

// One workgroup per (row, kv head) for more blocks: CH neighbouring ones a thread in
// registers (ONCE: NT x CH hold them all; else they are read again in each step).  T is
// found by up to four histograms of 8 bits, in LDS; a step's counts need one barrier.
// Against the bisection above with 1,024 threads, one row of 130,001 keys in blocks of
// 16 17.0 us, 32 rows of 1,024-4,096 blocks 19.4.
template <int NT, int CH, bool ONCE>
__global__ void __launch_bounds__(NT) select_kernel(SelectArgs a) {
  constexpr int NW = NT / 64;
  static_assert(CH % 4 == 0 && NW <= 16, "16-byte loads, a lane per wave");
  __shared__ __attribute__((aligned(16))) uint32_t hist[4][256];
  __shared__ uint32_t sums[2][2][16];
  const SelectRow r = select_row(a, blockIdx.x);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = a.width, nb = r.nb;
  if (nb <= K) {
    for (int j = tid; j < K; j += NT) r.out[j] = j < nb ? j : -1;
    return;
  }
  const int rounds = ONCE ? 1 : (nb + NT * CH - 1) / (NT * CH);
  uint32_t keys[CH];
  const auto load = [&](int i) {                          // blocks (i NT + tid) CH ..
    const int b0 = (i * NT + tid) * CH;
#pragma unroll
    for (int c = 0; c < CH; c += 4) {
      const u32x4 w = ld16(r.scores + (b0 + c < nb ? b0 + c : 0));    // rows are padded to 4
#pragma unroll
      for (int e = 0; e < 4; ++e) keys[c + e] = score_key(a, r, b0 + c + e, w[e]);
    }
  };
  const auto candidate = [](uint32_t k) { return k - 1u < 0xfffffffeu; };
  for (int j = tid; j < 4 * 256; j += NT) hist[j >> 8][j & 255] = 0u;
  if (ONCE) load(0);
  // the candidates' range
  uint32_t hi = 0u, nlo = 0u;
  for (int i = 0; i < rounds; ++i) {
    if (!ONCE) load(i);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      hi = max(hi, candidate(keys[c]) ? keys[c] : 0u);
      nlo = max(nlo, candidate(keys[c]) ? ~keys[c] : 0u);
    }
  }
  hi = wave_max(hi);
  nlo = wave_max(nlo);
  if (lane == 0) {
    sums[0][0][wave] = hi;
    sums[0][1][wave] = nlo;
  }
  __syncthreads();
  uint32_t take_from = 0xffffffffu;                       // keys above are taken, and `equal` ones of those equal
  int equal = K;
  if (K > a.first + a.recent) {
    hi = wave_max(sums[0][0][lane % NW]);
    const uint32_t lo = ~wave_max(sums[0][1][lane % NW]);
    int bit = __builtin_amdgcn_readfirstlane(hi == lo ? -1 : 31 - __clz((int)(hi ^ lo)));
    uint32_t T = bit < 0 ? hi : hi >> bit >> 1 << bit << 1;
    int above = a.first + a.recent;                       // keys above T's prefix
    bool exact = false;                                   // all keys with the prefix are taken
    for (int p = 0; bit >= 0 && !exact; ++p) {
      const int w = min(8, bit + 1), shift = bit + 1 - w;
      for (int i = 0; i < rounds; ++i) {
        if (!ONCE) load(i);
#pragma unroll
        for (int c = 0; c < CH; ++c)
          if (candidate(keys[c]) && (keys[c] ^ T) >> bit >> 1 == 0u) atomicAdd(&hist[p][(keys[c] >> shift) & ((1u << w) - 1)], 1u);
      }
      __syncthreads();
      // lane l: bins 4 l .. 4 l + 3 and the counts of all bins above them
      const u32x4 n = *reinterpret_cast<const u32x4*>(&hist[p][4 * lane]);
      uint32_t suffix = n[0] + n[1] + n[2] + n[3];
#pragma unroll
      for (int s = 1; s < 64; s *= 2) {
        const uint32_t y = (uint32_t)__shfl_down((int)suffix, s, 64);
        suffix += lane + s < 64 ? y : 0u;
      }
      uint32_t over = suffix - (n[0] + n[1] + n[2] + n[3]);   // keys in higher lanes' bins
      // the highest bin that reaches K
      int bin = -1;
      uint32_t bin_over = 0u, bin_n = 0u;
#pragma unroll
      for (int e = 3; e >= 0; --e) {
        if (bin < 0 && above + over + n[e] >= (uint32_t)K) {
          bin = 4 * lane + e;
          bin_over = over;
          bin_n = n[e];
        }
        over += n[e];
      }
      const int at = 63 - __clzll((long long)__builtin_amdgcn_ballot_w64(bin >= 0));
      bin = __builtin_amdgcn_readlane(bin, at);
      above += __builtin_amdgcn_readlane((int)bin_over, at);
      T |= (uint32_t)bin << shift;
      exact = above + __builtin_amdgcn_readlane((int)bin_n, at) == K;
      bit -= w;
    }
    take_from = exact ? max(T, 1u) - 1u : T;              // blocks' keys are above 0
    equal = exact ? 0 : K - above;
  }
  // places in block order: the threads' counts, of keys above and of equal ones, summed
  // up over the threads before
  int at = 0, eq_at = 0;
  for (int i = 0; i < rounds; ++i) {
    if (!ONCE) load(i);
    uint32_t gt = 0u, eq = 0u;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      gt += keys[c] > take_from;
      eq += keys[c] == take_from;
    }
    uint32_t g = gt, q = eq;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const uint32_t y = (uint32_t)__shfl_up((int)g, s, 64), z = (uint32_t)__shfl_up((int)q, s, 64);
      g += lane >= s ? y : 0u;
      q += lane >= s ? z : 0u;
    }
    uint32_t (*const sm)[16] = sums[(i + 1) & 1];
    if (lane == 63) {
      sm[0][wave] = g;
      sm[1][wave] = q;
    }
    __syncthreads();
    int place = at + (int)(g - gt), eq_place = eq_at + (int)(q - eq);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      place += w < wave ? (int)sm[0][w] : 0;
      eq_place += w < wave ? (int)sm[1][w] : 0;
      at += (int)sm[0][w];
      eq_at += (int)sm[1][w];
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const bool is_eq = keys[c] == take_from;
      if (keys[c] > take_from || (is_eq && eq_place < equal)) r.out[place + min(eq_place, equal)] = (i * NT + tid) * CH + c;
      place += keys[c] > take_from;
      eq_place += is_eq;
    }
  }
}

template <typename QT>
static hipError_t launch_scores_t(const SelectArgs& a, int hw, dim3 grid, hipStream_t st) {
  const dim3 block(64 * kScoreWaves);
  const int nk = (2 * a.head_dim + 63) / 64;
  const auto go = [&](auto n, auto gp, auto pass) {
    constexpr int NK = decltype(n)::value, GP = decltype(gp)::value;
    constexpr bool PASSES = decltype(pass)::value;
    constexpr int RT = PASSES || NK == 8 ? 1 : kScoreRowTiles;
    if (RT == 1 || a.row_tiles == 1) hipLaunchKernelGGL((block_scores_kernel<QT, NK, GP, 1, PASSES>), grid, block, 0, st, a, hw);
    else hipLaunchKernelGGL((block_scores_kernel<QT, NK, GP, RT, PASSES>), grid, block, 0, st, a, hw);
  };
  const auto by_group = [&](auto n) {
    const int G = a.num_q_heads / a.num_kv_heads;
    if (G == 1) go(n, std::integral_constant<int, 1>(), std::false_type());
    else if (G == 2) go(n, std::integral_constant<int, 2>(), std::false_type());
    else if (G <= 4) go(n, std::integral_constant<int, 4>(), std::false_type());
    else if (G <= 8) go(n, std::integral_constant<int, 8>(), std::false_type());
    else if (G <= 16) go(n, std::integral_constant<int, 16>(), std::false_type());
    else go(n, std::integral_constant<int, 16>(), std::true_type());
  };
  if (nk <= 2) by_group(std::integral_constant<int, 2>());
  else if (nk <= 4) by_group(std::integral_constant<int, 4>());
  else by_group(std::integral_constant<int, 8>());
  return hipGetLastError();
}

hipError_t launch_select_blocks(const SelectArgs& a, hipStream_t st) {
  if (a.n_rows == 0) return hipSuccess;
  const int64_t units = (int64_t)a.n_rows * a.num_kv_heads;
  if (units > INT32_MAX) return hipErrorInvalidValue;
  if (a.n_items > 0) {
    const int hw = score_heads(a.num_kv_heads);
    const int64_t wgs = (int64_t)a.n_items * (a.num_kv_heads / hw);
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    hipError_t e = hipErrorInvalidValue;
    const dim3 grid((unsigned)wgs);
    switch (a.dtype) {
      case kF32: e = launch_scores_t<float>(a, hw, grid, st); break;
      case kBF16: e = launch_scores_t<__bf16>(a, hw, grid, st); break;
      case kF16: e = launch_scores_t<_Float16>(a, hw, grid, st); break;
      default: break;
    }
    if (e != hipSuccess) return e;
  }
  const dim3 waves((unsigned)((units + kWaveSelects - 1) / kWaveSelects)), wblock(64 * kWaveSelects);
  const dim3 grid((unsigned)units);
  if (a.max_blocks <= 8 * 64) hipLaunchKernelGGL(select_wave_kernel<8>, waves, wblock, 0, st, a, (int)units);
  else if (a.max_blocks <= 256 * 8) hipLaunchKernelGGL((select_kernel<256, 8, true>), grid, dim3(256), 0, st, a);
  else if (a.max_blocks <= 1024 * 8) hipLaunchKernelGGL((select_kernel<1024, 8, true>), grid, dim3(1024), 0, st, a);
  else hipLaunchKernelGGL((select_kernel<1024, 8, false>), grid, dim3(1024), 0, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------- tiles of prompt rows
// For each (tile, kv head) the blocks that one of its rows selected, in order, each with
// a bit per row: a workgroup marks them in LDS, kTileWindow blocks of the sequence at a
// time, and writes the marked ones one after another.  A row's list counts up to its
// first entry out of order (selected_blocks).
constexpr int kTileThreads = 512;
constexpr int kTileWindow = 4096;
__global__ void __launch_bounds__(kTileThreads) tile_blocks_kernel(AttnArgs a) {
  constexpr int NW = kTileThreads / 64, PER = kTileWindow / kTileThreads;
  __shared__ unsigned long long mark[kTileWindow];
  __shared__ int len[64], own[64], sums[2][NW];
  const int ti = blockIdx.x / a.num_kv_heads, kvh = blockIdx.x - ti * a.num_kv_heads;
  const SparseTile st = a.sparse_tiles[ti];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = a.sel_width;
  if (tid < st.nrows) {
    len[tid] = K;
    own[tid] = (int)div_bs((uint32_t)a.tile_rows[st.row0 + tid].pos, a.block_magic, a.block_shift);
  }
  const auto list = [&](int r) { return a.selected + ((int64_t)a.tile_rows[st.row0 + r].row * a.num_kv_heads + kvh) * K; };
  __syncthreads();
  // a wave a row
  for (int r = wave; r < st.nrows; r += NW) {
    const int32_t* sel = list(r);
    int n = K;
    for (int j = lane; j < K; j += 64) {
      const int x = sel[j], before = j > 0 ? sel[j - 1] : -1;
      if (x <= before || x < 0 || x > own[r]) n = min(n, j);
    }
#pragma unroll
    for (int s = 1; s < 64; s *= 2) n = min(n, __shfl_xor(n, s, 64));
    if (lane == 0) len[r] = n;
  }
  const int last = own[st.nrows - 1];                    // rows are in the order of their positions
  SelectedBlock* out = a.tile_entries + (int64_t)blockIdx.x * a.tile_capacity;
  int at = 0, flip = 0;
  for (int w0 = 0; w0 <= last; w0 += kTileWindow) {
    for (int j = tid; j < kTileWindow; j += kTileThreads) mark[j] = 0ull;
    __syncthreads();
    for (int r = wave; r < st.nrows; r += NW) {
      const int32_t* sel = list(r);
      for (int j = lane; j < len[r]; j += 64) {
        const int x = sel[j] - w0;
        if (x >= 0 && x < kTileWindow) atomicOr(&mark[x], 1ull << r);
      }
    }
    __syncthreads();
    // a thread's neighbouring blocks; their places from the threads before
    unsigned long long m[PER];
    int n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      m[i] = mark[tid * PER + i];
      n += m[i] != 0;
    }
    int upto = n;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const int y = __shfl_up(upto, s, 64);
      upto += lane >= s ? y : 0;
    }
    if (lane == 63) sums[flip][wave] = upto;
    __syncthreads();
    int place = at + upto - n;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      place += w < wave ? sums[flip][w] : 0;
      at += sums[flip][w];
    }
    flip ^= 1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (m[i] == 0) continue;
      const int b = w0 + tid * PER + i;
      const uint32_t blk = (uint32_t)a.block_table[(int64_t)st.seq * a.block_table_stride + b];
      if (place < a.tile_capacity)
        out[place] = SelectedBlock{m[i], b, blk < (uint64_t)a.num_blocks ? (int32_t)blk : 0};   // never outside the pool
      ++place;
    }
  }
  // the last row's own block, if any row selected it, ends at that row's key: nothing
  // behind it is read
  if (tid == 0) {
    const int keys = min(at, a.tile_capacity) * a.block_size, pos = a.tile_rows[st.row0 + st.nrows - 1].pos;
    const bool ends = mark[last % kTileWindow] != 0;
    a.tile_keys[blockIdx.x] = keys - (ends ? (last + 1) * a.block_size - 1 - pos : 0);
  }
}
hipError_t launch_tile_blocks(const AttnArgs& a, hipStream_t st) {
  const int64_t units = (int64_t)a.n_sparse_tiles * a.num_kv_heads;
  if (units > INT32_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL(tile_blocks_kernel, dim3((unsigned)units), dim3(kTileThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace gllm
