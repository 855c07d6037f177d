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
  __syncthreads();
  if (g < kg) {
    for (int t = g; t < bb.n; t += kg) {
      float x[8];
      if constexpr (std::is_same<KV, kv4>::value) {
        const uint8_t* rec = (const uint8_t*)a.k_cache + (int64_t)blk * a.cache_slot_stride + (int64_t)(h0 + hh) * a.kv4_record;
        load8_kv<KV, QT>(rec + t * (D / 2), d, rec + (int64_t)a.block_size * (D / 2) + t * (D / 32), x);
      } else {
        const KV* row = (const KV*)a.k_cache + ((int64_t)blk * a.block_size + t) * a.cache_slot_stride + (int64_t)(h0 + hh) * D;
        load8_kv<KV, QT>(row, d, nullptr, x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = fminf(lo[i], x[i]);
        hi[i] = fmaxf(hi[i], x[i]);
        m = max(m, magnitude(x[i]));                     // a NaN's bits are above infinity's
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
// One workgroup per (tile of query rows, chunk of kScoreGroups x 16 blocks); wave w
// takes the kv heads w, w + 4, ...  A column of the MFMA is a (row of the tile, head of
// the group) pair, n = row x Gp + g with Gp = G rounded up to a power of two, so a
// tile's rows share the bounds they load; more than 16 heads go by in passes.  Lane
// (n, grp) loads bytes 64 s + 16 grp .. + 15 of block n's [lo | hi], every load of a head
// in flight at once; the codes of q lie in the same order.  HBM- or L2-bound by the
// bounds of long sequences.
constexpr int kScoreGroups = 4;
constexpr int kScoreWaves = 4;
template <typename QT, int NK>
__global__ void __launch_bounds__(64 * kScoreWaves) block_scores_kernel(SelectArgs a, int gp_log, int chunks) {
  const int tile = blockIdx.x / chunks, chunk = blockIdx.x - tile * chunks;
  const ScoreTile tl = a.tiles[a.tile0 + tile];
  const int b0 = chunk * kScoreGroups * 16;
  if (b0 >= tl.nblocks) return;
  const int lane = threadIdx.x & 63, n = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int D = a.head_dim, G = a.num_q_heads / a.num_kv_heads, Hkv = a.num_kv_heads;
  const int gp = 1 << gp_log, ri = n >> gp_log, g0 = n & (gp - 1);
  const bool row_ok = ri < tl.nrows;
  const int row = a.rows[tl.row0 + (row_ok ? ri : 0)].row;
  const int passes = (G + 15) / 16;
  // the lane's blocks, one of each group: their records
  const uint8_t* rec[kScoreGroups];
#pragma unroll
  for (int u = 0; u < kScoreGroups; ++u) {
    const int b = min(b0 + 16 * u + n, tl.nblocks - 1);
    uint32_t blk = (uint32_t)a.block_table[(int64_t)tl.seq * a.block_table_stride + b];
    if (blk >= (uint64_t)a.num_blocks) blk = 0;          // never address outside the pool
    rec[u] = a.bounds + (int64_t)blk * a.bounds_stride;
  }
  for (int h = wave; h < Hkv; h += kScoreWaves) {
    u32x4 box[kScoreGroups][NK];
    int exps[kScoreGroups];
#pragma unroll
    for (int u = 0; u < kScoreGroups; ++u) {
#pragma unroll
      for (int s = 0; s < NK; ++s) box[u][s] = ld16(rec[u] + h * 2 * D + min(64 * s + 16 * grp, 2 * D - 16));
      exps[u] = rec[u][Hkv * 2 * D + h];
    }
    int best[kScoreGroups][4];
#pragma unroll
    for (int u = 0; u < kScoreGroups; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) best[u][j] = INT32_MIN;
    // one power of two for all heads of the group
    uint32_t m = 0u;
    float x[2 * NK][8];
    const auto load_q = [&](int p) {
      const int g = min(16 * p + g0, G - 1);
      const QT* qp = (const QT*)a.q + (int64_t)row * a.q_row_stride + (int64_t)(h * G + g) * D;
#pragma unroll
      for (int s = 0; s < 2 * NK; ++s) {
        const int k = 64 * (s / 2) + 16 * grp + 8 * (s % 2);
        load8<QT>(qp + min(k < D ? k : k - D, D - 8), x[s]);
      }
    };
    for (int p = 0; p < passes; ++p) {
      load_q(p);
#pragma unroll
      for (int s = 0; s < 2 * NK; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, magnitude(x[s][i]));
    }
    m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
    m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
    for (int s = 1; s < gp; s *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, s, 64));
    const float inv = m > kCodeMax ? 0.f : pow2f(-code_exponent(m));
    for (int p = 0; p < passes; ++p) {
      if (passes > 1) load_q(p);
      u32x4 qb[NK];
#pragma unroll
      for (int s = 0; s < 2 * NK; ++s) {
        const int k = 64 * (s / 2) + 16 * grp + 8 * (s % 2);
        const bool none = !row_ok || k >= 2 * D || m > kCodeMax;
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float c = __builtin_rintf(x[s][i] * inv);
          const float half = k < D ? fminf(c, 0.f) : fmaxf(c, 0.f);     // lo takes the negative codes
          w[i / 4] |= (uint32_t)(uint8_t)(int8_t)(int)half << (8 * (i % 4));
        }
        qb[s / 2][2 * (s % 2)] = none ? 0u : w[0];
        qb[s / 2][2 * (s % 2) + 1] = none ? 0u : w[1];
      }
#pragma unroll
      for (int u = 0; u < kScoreGroups; ++u) {
        i32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NK; ++s)
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, box[u][s]), __builtin_bit_cast(i32x4, qb[s]), acc, 0, 0, 0);
        const bool real = 16 * p + g0 < G;
#pragma unroll
        for (int j = 0; j < 4; ++j) best[u][j] = max(best[u][j], real ? acc[j] : INT32_MIN);
      }
    }
#pragma unroll
    for (int u = 0; u < kScoreGroups; ++u) {
      f32x4 sc;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int v = best[u][j];
        for (int s = 1; s < gp; s *= 2) v = max(v, __shfl_xor(v, s, 64));
        const int e = __shfl(exps[u], 4 * grp + j, 64);   // lane 4 grp + j holds block 4 grp + j's
        // bytes that no writer leaves are limited, so that the score stays a number
        sc[j] = e == kOpen ? -kNegInf : (float)v * pow2f(min(max(e - 128, -100), 100));
      }
      if (row_ok && g0 == 0) {
        const int b = b0 + 16 * u + 4 * grp;
        float* sp = a.scores + ((int64_t)(tl.row0 + ri - a.row0) * Hkv + h) * a.score_stride + b;
        if (b < a.score_stride) *reinterpret_cast<f32x4*>(sp) = sc;   // rows are padded to 4
      }
    }
  }
}

// ---------------------------------------------------------------- selection
// One workgroup per (row, kv head): the width-th largest key by bisection over its bits
// (a count of the keys above a candidate a step, until a candidate keeps exactly as
// many), then the blocks above it and the first of those equal to it, in order.  Keys
// are the scores as unsigned integers of the same order; blocks that are always taken
// have the largest.  NR > 0: up to NR x 512 blocks, held in registers; 0: any number,
// read again in each step.
constexpr int kSelectThreads = 512;
template <int NR>
__global__ void __launch_bounds__(kSelectThreads) select_kernel(SelectArgs a) {
  constexpr int NW = kSelectThreads / 64;
  __shared__ int cnt[2][NW];
  __shared__ int cnt2[2][NW];
  const int ri = blockIdx.x / a.num_kv_heads, h = blockIdx.x - ri * a.num_kv_heads;
  const SparseRow sr = a.rows[a.row0 + ri];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = (int)div_bs((uint32_t)sr.pos, a.block_magic, a.block_shift) + 1;
  int32_t* out = a.selected + ((int64_t)sr.row * a.num_kv_heads + h) * a.width;
  const int K = a.width;
  if (nb <= K) {
    for (int j = tid; j < K; j += kSelectThreads) out[j] = j < nb ? j : -1;
    return;
  }
  const float* sp = a.scores + ((int64_t)ri * a.num_kv_heads + h) * a.score_stride;
  const auto key_at = [&](int b) -> uint32_t {
    if (b >= nb) return 0u;
    if (b < a.first || b >= nb - a.recent) return 0xffffffffu;
    const uint32_t u = __float_as_uint(sp[b]);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
  };
  uint32_t keys[NR > 0 ? NR : 1];
  if constexpr (NR > 0) {
#pragma unroll
    for (int i = 0; i < NR; ++i) keys[i] = key_at(tid + i * kSelectThreads);
  }
  const int rounds = NR > 0 ? NR : (nb + kSelectThreads - 1) / kSelectThreads;
  int flip = 0;
  // keys of the workgroup that are at least c
  const auto count = [&](uint32_t c) {
    int n = 0;
    if constexpr (NR > 0) {
#pragma unroll
      for (int i = 0; i < NR; ++i) n += __popcll(__builtin_amdgcn_ballot_w64(keys[i] >= c));
    } else {
      for (int i = 0; i < rounds; ++i) n += __popcll(__builtin_amdgcn_ballot_w64(key_at(tid + i * kSelectThreads) >= c));
    }
    if (lane == 0) cnt[flip][wave] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) n += cnt[flip][w];
    flip ^= 1;                                            // the next count writes the other row
    return n;
  };
  uint32_t T = 0u;
  int above = 0;                                          // keys >= T + (the bit just refused)
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = T | (1u << bit);
    const int n = count(c);
    if (n >= K) {
      T = c;
      if (n == K) break;                                  // exactly these
    }
  }
  above = T == 0xffffffffu ? 0 : count(T + 1);            // keys > T; of those equal to T the first K - above
  int eq_left = K - above, at = 0;
  for (int i = 0; i < rounds; ++i) {
    uint32_t k = 0u;
    if constexpr (NR > 0) {
#pragma unroll
      for (int r = 0; r < NR; ++r) k = i == r ? keys[r] : k;
    } else {
      k = key_at(tid + i * kSelectThreads);
    }
    const uint64_t eq = __builtin_amdgcn_ballot_w64(k == T), gt = __builtin_amdgcn_ballot_w64(k > T);
    if (lane == 0) {
      cnt[flip][wave] = __popcll(gt);
      cnt2[flip][wave] = __popcll(eq);
    }
    __syncthreads();
    // equal keys are taken while eq_left lasts: those before this wave's, and its own
    int eq_before = 0, pos = at;
    int eq_all = 0, gt_all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < wave) {
        pos += cnt[flip][w];
        eq_before += cnt2[flip][w];
      }
      gt_all += cnt[flip][w];
      eq_all += cnt2[flip][w];
    }
    const uint64_t below = (1ull << lane) - 1;
    const int eq_mine = eq_before + __popcll(eq & below);
    const bool take = k > T || (k == T && eq_mine < eq_left);
    pos += __popcll(gt & below) + min(eq_mine, eq_left);
    if (take) out[pos] = tid + i * kSelectThreads;
    at += gt_all + min(eq_all, eq_left);
    eq_left -= min(eq_all, eq_left);
    flip ^= 1;
  }
}

template <typename QT>
static hipError_t launch_scores_t(const SelectArgs& a, int gp_log, int chunks, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.n_tiles * chunks)), block(64 * kScoreWaves);
  const int nk = (2 * a.head_dim + 63) / 64;
  if (nk <= 2) hipLaunchKernelGGL((block_scores_kernel<QT, 2>), grid, block, 0, st, a, gp_log, chunks);
  else if (nk <= 4) hipLaunchKernelGGL((block_scores_kernel<QT, 4>), grid, block, 0, st, a, gp_log, chunks);
  else hipLaunchKernelGGL((block_scores_kernel<QT, 8>), grid, block, 0, st, a, gp_log, chunks);
  return hipGetLastError();
}

hipError_t launch_select_blocks(const SelectArgs& a, hipStream_t st) {
  if (a.n_rows == 0) return hipSuccess;
  if (a.n_tiles > 0) {
    const int G = a.num_q_heads / a.num_kv_heads;
    int gp_log = 0;
    while ((1 << gp_log) < G && gp_log < 4) ++gp_log;
    const int chunks = (a.max_blocks + kScoreGroups * 16 - 1) / (kScoreGroups * 16);
    if ((int64_t)a.n_tiles * chunks > INT32_MAX) return hipErrorInvalidValue;
    hipError_t e = hipErrorInvalidValue;
    switch (a.dtype) {
      case kF32: e = launch_scores_t<float>(a, gp_log, chunks, st); break;
      case kBF16: e = launch_scores_t<__bf16>(a, gp_log, chunks, st); break;
      case kF16: e = launch_scores_t<_Float16>(a, gp_log, chunks, st); break;
      default: break;
    }
    if (e != hipSuccess) return e;
  }
  if ((int64_t)a.n_rows * a.num_kv_heads > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(a.n_rows * a.num_kv_heads)), block(kSelectThreads);
  if (a.max_blocks <= 4 * kSelectThreads) hipLaunchKernelGGL(select_kernel<4>, grid, block, 0, st, a);
  else if (a.max_blocks <= 16 * kSelectThreads) hipLaunchKernelGGL(select_kernel<16>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(select_kernel<0>, grid, block, 0, st, a);
  return hipGetLastError();
}

}  // namespace gllm
