// Rotary positions + paged KV write without a cos/sin table, and everything
// that writes or reads back the rows of a 4-bit cache (format: common.h).
//
// Rotary: the token at position p turns pair i by p f_i (f_i in radians per
// position, any schedule of frequencies), with cos and sin times a factor:
// [x1 c - x2 s, x1 s + x2 c] over pairs (i, i + R/2) or (2i, 2i + 1) of the first
// R dims; the rest of the head passes.  No counterpart in the reference, whose
// table is one of half pairs over the whole head at a single theta.
//
// The angle is one fp64 product: at position 10^6 an fp32 product is off by
// 0.06 rad.  It is reduced by quarter turns and sin and cos are their Taylor
// series on |r| <= pi/4 (below 2^-53 of the result), all in fp64, R/2 of them a
// token, shared by its heads.  q is rotated in fp32 and rounded once to the
// model dtype; k in fp64, and rounded once to the cache dtype: values that an
// 8- or 4-bit cache rounds come next to a border often enough for an fp32
// product to choose the other code (fp64 FMAs run at the fp32 rate here).
//
// HBM-bound: every element is read once and written once.  One wave per token
// (per part of one where tokens are few); a lane keeps its 8 dims across the
// heads, so its eight (cos, sin) stay in registers.
#include <type_traits>

#include "common.h"
#include "generic.h"
#include "launch.h"

namespace gllm {

// 8 elements at p as floats
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  if constexpr (std::is_same<T, float>::value) {
    const u32x4 a = ld16(p), b = ld16(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __uint_as_float(a[i]);
      v[4 + i] = __uint_as_float(b[i]);
    }
  } else {
    unpack8<T>(ld16(p), v);
  }
}
template <typename S>
__device__ __forceinline__ void store8(S* p, const float* v) {
  if constexpr (std::is_same<S, float>::value) {
    st16(p, u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
    st16(p + 4, u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
  } else if constexpr (std::is_same<S, fp8e4m3>::value) {
    st8(p, u32x2{pack_fp8x4(v[0], v[1], v[2], v[3]), pack_fp8x4(v[4], v[5], v[6], v[7])});
  } else {
    st16(p, pack8<S>(v));
  }
}

// fp64 -> fp32 with the last bit set where bits were lost (round to odd): a
// second rounding, to 16, 8 or 4 bits, then gives what one from fp64 gives.
__device__ __forceinline__ float to_odd(double d) {
  const float f = (float)d;
  const double r = d - (double)f;
  uint32_t u = __float_as_uint(f);
  // f is nearest: the other neighbour is one step towards d; NaN and infinity stay
  if (r != 0.0 && !(u & 1u) && __builtin_isfinite(f)) u += (r > 0.0) == (f > 0.f || (f == 0.f && r > 0.0)) ? 1u : ~0u;
  if (f == 0.f && r < 0.0) u = 0x80000001u;
  return __uint_as_float(u);
}

// c = m cos a, s = m sin a.  a = n pi/2 + r with |r| <= pi/4: n hi is exact in the
// FMA, lo is what fp64 drops of pi/2.
__device__ __forceinline__ void sincos64(double a, double m, double* c, double* s) {
  constexpr double kHi = 1.57079632679489655800, kLo = 6.12323399573676603587e-17, kInv = 0.63661977236758134308;
  const double n = __builtin_rint(a * kInv);
  const double r = __builtin_fma(-n, kLo, __builtin_fma(-n, kHi, a));
  const double z = r * r;
  // Taylor: sin r = r (1 - z/3! + ... - z^7/15!), cos r = 1 - z/2! + ... + z^8/16!
  double ps = -1.0 / 1307674368000.0, pc = 1.0 / 20922789888000.0;
  ps = __builtin_fma(ps, z, 1.0 / 6227020800.0);
  ps = __builtin_fma(ps, z, -1.0 / 39916800.0);
  ps = __builtin_fma(ps, z, 1.0 / 362880.0);
  ps = __builtin_fma(ps, z, -1.0 / 5040.0);
  ps = __builtin_fma(ps, z, 1.0 / 120.0);
  ps = __builtin_fma(ps, z, -1.0 / 6.0);
  pc = __builtin_fma(pc, z, -1.0 / 87178291200.0);
  pc = __builtin_fma(pc, z, 1.0 / 479001600.0);
  pc = __builtin_fma(pc, z, -1.0 / 3628800.0);
  pc = __builtin_fma(pc, z, 1.0 / 40320.0);
  pc = __builtin_fma(pc, z, -1.0 / 720.0);
  pc = __builtin_fma(pc, z, 1.0 / 24.0);
  pc = __builtin_fma(pc, z, -0.5);
  const double sr = __builtin_fma(ps * z, r, r), cr = __builtin_fma(pc, z, 1.0);
  const int q = (int)(int64_t)n & 3;           // quarter turns
  const double cc = q & 1 ? sr : cr, ss = q & 1 ? cr : sr;
  *c = m * (q == 1 || q == 2 ? -cc : cc);
  *s = m * (q >= 2 ? -ss : ss);
}

// The largest of x over the four lanes of a quad (non-negative floats as bits).
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, false));   // lanes 1 0 3 2
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, false));   // lanes 2 3 0 1
}

// 8 of the 32 values of a block (the quad of lanes holds them all) as codes;
// *byte the block's scale.  T: the model dtype, which the rows are read in.  An
// fp16 model's values stop at +-6 x 2^13: the next larger value that a block can
// stand for, 4 x 2^14, is infinite in fp16 (values round to it from 57,344 on).
template <typename T>
__device__ __forceinline__ uint32_t encode4(float* v, uint32_t* byte) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
  amax = quad_max(amax);
  if (amax >= 0x7f800000u) {             // an infinity or NaN
    *byte = 255u;
    return 0u;
  }
  if constexpr (std::is_same<T, _Float16>::value) {
    constexpr float top = kKv4MaxF16;
    amax = min(amax, __float_as_uint(top));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_amdgcn_fmed3f(v[i], -top, top);
  }
  // the least e with amax < 7 x 2^e: 7 = 1.75 x 4, so a mantissa from 1.75 on
  // carries into the exponent here
  const uint32_t e = (amax + 0x00200000u) >> 23;
  *byte = e > 3u ? e - 2u : 1u;
  const float scale = __uint_as_float(*byte << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}

constexpr int kRotWaves = 4;        // waves per workgroup
// LDS place of a pair's (cos, sin): a gap after every eight, so that lanes
// eight pairs apart read different banks
__device__ __forceinline__ int pair_at(int i) { return i + (i >> 3); }
constexpr int kRotPairs = 128 + 16;  // places of the most pairs of a head (head_dim 256)

// TABLE: cos / sin rows in the model dtype and every op rounded to it, half
// pairs over the whole head: rope_kv_write's arithmetic
// (gllm/model/layers/attention.py:91-118).
template <typename T, typename KV, bool TABLE>
__global__ void __launch_bounds__(64 * kRotWaves) rotary_write_kernel(RotaryWriteArgs a) {
  __shared__ double cs[TABLE ? 1 : kRotWaves][TABLE ? 1 : kRotPairs][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int D = a.head_dim, R = a.rotary_dim, half = R / 2;
  const int cpd = D / 8;                          // 8-dim chunks of a head
  const int hpi = 64 / cpd;                       // heads of one pass of the wave
  const int ch = lane % cpd, hl = lane / cpd;     // the lane's chunk and head of the pass
  const int d0 = 8 * ch;
  const int nq = a.q_out ? (a.num_q_heads + hpi - 1) / hpi : 0;
  // the pair that dim d belongs to (-1: it passes), and the sign of its partner's product
  auto pair_of = [&](int d) { return d >= R ? -1 : (a.interleaved ? d / 2 : (d < half ? d : d - half)); };
  auto flip = [&](int d) { return (a.interleaved ? !(d & 1) : d < half) ? -1.f : 1.f; };
  const int nk = a.k ? (a.num_kv_heads + hpi - 1) / hpi : 0;
  const int part = blockIdx.y;
  const int64_t tok = (int64_t)blockIdx.x * kRotWaves + wave;   // no loop over tokens: its invariants would fill the registers
  if (tok >= a.num_tokens) return;
  if (a.query_lens) {                           // padded rows are skipped whole
    const int64_t b = tok / a.tokens_per_seq;
    if (tok - b * a.tokens_per_seq >= a.query_lens[b]) return;
  }
  int64_t slot = -1;
  if (a.k) slot = a.slot_mapping[tok];
  const bool kv_ok = slot >= 0 && slot < a.num_slots;   // never address outside the pool
  int64_t at = slot * a.cache_slot_stride;              // the row's place in the caches
  int64_t sc_at = 0;                                    // 4-bit: its scales'
  if constexpr (std::is_same<KV, kv4>::value) {
    const int64_t blk = kv_ok ? slot / a.block_size : 0, off = slot - blk * a.block_size;
    at = blk * a.cache_slot_stride + off * (D / 2);
    sc_at = blk * a.cache_slot_stride + (int64_t)a.block_size * (D / 2) + off * (D / 32);
  }

  // cos and sin of the lane's 8 dims: q's in registers, k's (fp64) stay in LDS
  float c32[8], s32[8];
  if constexpr (TABLE) {
    const int64_t row = a.rope_rows ? a.rope_rows[tok] : tok;
    const int j = d0 < half ? d0 : d0 - half;
    load8<T>((const T*)a.cos + row * a.rope_row_stride + j, c32);
    load8<T>((const T*)a.sin + row * a.rope_row_stride + j, s32);
  } else {
    const double p = (double)a.positions[tok];
    __builtin_amdgcn_wave_barrier();
    for (int i = lane; i < half; i += 64) {
      double ci, si;
      sincos64(p * a.freq[i], a.factor, &ci, &si);
      cs[wave][pair_at(i)][0] = ci;
      cs[wave][pair_at(i)][1] = si;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // the wave's own LDS, in order
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pr = pair_of(d0 + i);
      c32[i] = pr < 0 ? 1.f : (float)cs[wave][pair_at(pr)][0];
      s32[i] = pr < 0 ? 0.f : flip(d0 + i) * (float)cs[wave][pair_at(pr)][1];
    }
  }

  // the row's 8 dims and their partners
  auto pair8 = [&](const T* row, float* x, float* y) {
    load8<T>(row + d0, x);
    if (!TABLE && a.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
    } else if (TABLE || half % 8 == 0) {         // a chunk lies in one half
      const int dp = d0 < half ? d0 + half : (d0 < R ? d0 - half : d0);
      load8<T>(row + dp, y);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        y[i] = (float)row[d < half ? d + half : (d < R ? d - half : d)];
      }
    }
  };
  auto turn_ops = [&](const float* x, const float* y, float* o) {     // each op rounded to T
    const bool first = d0 < half;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float u0 = rnd<T>(__fmul_rn(x[i], c32[i])), v0 = rnd<T>(__fmul_rn(y[i], s32[i]));
      float u1 = rnd<T>(__fmul_rn(x[i + 1], c32[i + 1])), v1 = rnd<T>(__fmul_rn(y[i + 1], s32[i + 1]));
      if constexpr (std::is_same<T, _Float16>::value) opaque4(u0, v0, u1, v1);
      o[i] = rnd<T>(first ? __fsub_rn(u0, v0) : __fadd_rn(u0, v0));
      o[i + 1] = rnd<T>(first ? __fsub_rn(u1, v1) : __fadd_rn(u1, v1));
    }
  };

  for (int g = part; g < nq; g += gridDim.y) {
    const int h = g * hpi + hl;
    if (hl >= hpi || h >= a.num_q_heads) continue;
    float x[8], y[8];
    pair8((const T*)a.q + tok * a.q_row_stride + (int64_t)h * D, x, y);
    if constexpr (TABLE) {
      float o[8];
      turn_ops(x, y, o);
      store8<T>((T*)a.q_out + tok * a.q_out_row_stride + (int64_t)h * D + d0, o);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = d0 + i < R ? __builtin_fmaf(y[i], s32[i], x[i] * c32[i]) : x[i];
      store8<T>((T*)a.q_out + tok * a.q_out_row_stride + (int64_t)h * D + d0, x);
    }
  }
  if (!kv_ok) return;
  // the first of k's passes goes to the part after q's last, so that few parts have more than one
  for (int g = (part + gridDim.y - nq % gridDim.y) % gridDim.y; g < 2 * nk; g += gridDim.y) {
    const bool is_v = g >= nk;
    const int h = (is_v ? g - nk : g) * hpi + hl;
    if (hl >= hpi || h >= a.num_kv_heads) continue;
    float x[8], y[8];
    if (is_v) {
      load8<T>((const T*)a.v + tok * a.v_row_stride + (int64_t)h * D + d0, x);
    } else {
      pair8((const T*)a.k + tok * a.k_row_stride + (int64_t)h * D, x, y);
      if constexpr (TABLE) {
        float o[8];
        turn_ops(x, y, o);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = o[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int pr = pair_of(d0 + i);
          if (pr < 0) continue;
          const double c = cs[wave][pair_at(pr)][0], sn = cs[wave][pair_at(pr)][1] * (double)flip(d0 + i);
          const double d = __builtin_fma((double)y[i], sn, (double)x[i] * c);
          x[i] = std::is_same<KV, float>::value ? (float)d : to_odd(d);
        }
      }
    }
    void* const cache = is_v ? a.v_cache : a.k_cache;
    if constexpr (std::is_same<KV, kv4>::value) {
      uint8_t* const rec = (uint8_t*)cache + (int64_t)h * a.kv4_record;
      uint32_t byte;
      const uint32_t w = encode4<T>(x, &byte);
      *reinterpret_cast<uint32_t*>(rec + at + 4 * ch) = w;
      if ((ch & 3) == 0) rec[sc_at + ch / 4] = (uint8_t)byte;
    } else {
      store8<KV>((KV*)cache + at + (int64_t)h * D + d0, x);
    }
  }
}

// Rows of a 4-bit cache as values of T: one thread per 8 dims.
template <typename T>
__global__ void __launch_bounds__(256) kv4_values_kernel(Kv4ValuesArgs a) {
  const int D = a.head_dim, cpd = D / 8;
  const int per = a.num_kv_heads * cpd;
  const int64_t n = a.num_rows * per;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const int64_t row = e / per;
    const int rem = (int)(e - row * per), h = rem / cpd, ch = rem - h * cpd;
    const int64_t slot = a.slots[row];
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (slot >= 0 && slot < a.num_slots) {          // rows outside the pool: zeros
      const int64_t blk = slot / a.block_size, off = slot - blk * a.block_size;
      const uint8_t* rec = (const uint8_t*)a.cache + blk * a.block_stride + (int64_t)h * a.kv4_record;
      const uint32_t w = *reinterpret_cast<const uint32_t*>(rec + off * (D / 2) + 4 * ch);
      const float scale = __uint_as_float((uint32_t)rec[(int64_t)a.block_size * (D / 2) + off * (D / 32) + ch / 4] << 23);
      auto two = [&](auto x, int i) {
        v[i] = x[0];
        v[i + 1] = x[1];
      };
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), 0);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1), 2);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), 4);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3), 6);
    }
    store8<T>((T*)a.out + row * a.out_row_stride + (int64_t)h * D + 8 * ch, v);
  }
}

template <typename T>
static hipError_t launch_rotary_t(const RotaryWriteArgs& a, dim3 grid, hipStream_t st) {
  const dim3 block(64 * kRotWaves);
  if (a.cos) {
    hipLaunchKernelGGL((rotary_write_kernel<T, kv4, true>), grid, block, 0, st, a);
    return hipGetLastError();
  }
  switch (a.k ? a.kv_dtype : a.dtype) {
    case kF32: hipLaunchKernelGGL((rotary_write_kernel<T, float, false>), grid, block, 0, st, a); break;
    case kBF16: hipLaunchKernelGGL((rotary_write_kernel<T, __bf16, false>), grid, block, 0, st, a); break;
    case kF16: hipLaunchKernelGGL((rotary_write_kernel<T, _Float16, false>), grid, block, 0, st, a); break;
    case kFP8: hipLaunchKernelGGL((rotary_write_kernel<T, fp8e4m3, false>), grid, block, 0, st, a); break;
    case kMXFP4: hipLaunchKernelGGL((rotary_write_kernel<T, kv4, false>), grid, block, 0, st, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_rotary_write(const RotaryWriteArgs& a, int cus, hipStream_t st) {
  const int hpi = 64 / (a.head_dim / 8);
  const int passes = (a.q_out ? (a.num_q_heads + hpi - 1) / hpi : 0) + (a.k ? 2 * ((a.num_kv_heads + hpi - 1) / hpi) : 0);
  if (a.num_tokens == 0 || passes == 0) return hipSuccess;
  // few tokens: their passes go to several waves, up to two per SIMD
  const int64_t want = (int64_t)cus * 8 / a.num_tokens;
  const int parts = (int)(want < 1 ? 1 : (want > passes ? passes : want));
  const int64_t blocks = (a.num_tokens + kRotWaves - 1) / kRotWaves;
  if (blocks > 0x7fffffff / kRotWaves / 64) return hipErrorInvalidValue;   // the grid's threads
  const dim3 grid((unsigned)blocks, (unsigned)parts);
  switch (a.dtype) {
    case kF32: return launch_rotary_t<float>(a, grid, st);
    case kBF16: return launch_rotary_t<__bf16>(a, grid, st);
    case kF16: return launch_rotary_t<_Float16>(a, grid, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_kv4_values(const Kv4ValuesArgs& a, hipStream_t st) {
  const int64_t n = a.num_rows * a.num_kv_heads * (a.head_dim / 8);
  if (n == 0) return hipSuccess;
  int64_t blocks = (n + 255) / 256;
  if (blocks > 65536) blocks = 65536;
  const dim3 grid((unsigned)blocks), block(256);
  switch (a.dtype) {
    case kF32: hipLaunchKernelGGL((kv4_values_kernel<float>), grid, block, 0, st, a); break;
    case kBF16: hipLaunchKernelGGL((kv4_values_kernel<__bf16>), grid, block, 0, st, a); break;
    case kF16: hipLaunchKernelGGL((kv4_values_kernel<_Float16>), grid, block, 0, st, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace gllm
