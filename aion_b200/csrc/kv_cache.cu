// Quantized KV caches: rows are quantized as they are appended, logical steps are read back as values, and the
// projection's heads are normed, rotated and appended in one pass.
//
// A cache row of a head is D / 32 blocks of the weight formats: q8_0 (f16 scale, 32 int8) or q4_0 (f16 scale,
// 16 bytes of nibbles). The codes are those of aion_cuda_quantize, so this file is compiled without FMA
// contraction too. All three steps move each byte once and compute little: HBM bounds the large ones, the
// launch and one trip to memory the small ones.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "cache_geom.cuh"
#include "common.cuh"
#include "ptx.cuh"
#include "quant_device.cuh"

namespace aion {

namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;

// ---- the block quantizer, eight lanes to a block ------------------------------------------------
// Nearest whole number, halves away from zero, as the int conversion of roundf: the sum is cut off towards zero, so
// 0.5 minus an ulp stays below one. (One operation on the conversion unit instead of roundf's two.) NaN gives 0.
__device__ __forceinline__ int round_away(float r) { return __float2int_rz(__fadd_rz(r, copysignf(0.5f, r))); }

// v / s correctly rounded, for a divisor that many values share: y is its correctly rounded reciprocal, and the quotient
// v y is corrected twice by q + (v - s q) y with fused products (P. Markstein, Computation of elementary functions on
// the IBM RISC System/6000, 1990). The remainders are exact but where the quotient is far below one half.
__device__ __forceinline__ float quotient(float v, float s, float y) {
  float q = __fmul_rn(v, y);
  q = __fmaf_rn(__fmaf_rn(-s, q, v), y, q);
  return __fmaf_rn(__fmaf_rn(-s, q, v), y, q);
}

// Lane i of eight (i = lane & 7) holds values 4i .. 4i + 3 of a block. Returns the block's f16 scale and this
// lane's codes: q8_0 four bytes, q4_0 four nibbles. The same numbers as the block quantizer of quant.cu.
// All lanes of a warp call it together.
template <int DT>
__device__ __forceinline__ uint32_t quantize_4(const float (&v)[4], uint16_t* scale_bits) {
  float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
  amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 2));
  amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 4));
  uint32_t codes = 0;
  // Scales far from f32's ends, and from f16's lower one: every quotient is within half a code of the range, and none
  // has to be cut off.
  const bool plain = amax > 1e-2f && amax < 1e30f;
  if (DT == AION_CUDA_DTYPE_Q8_0) {
    float scale = 1.0f;
    if (plain) scale = quotient(amax, 127.0f, 1.0f / 127.0f);
    else if (amax != 0.0f) scale = __fdiv_rn(amax, 127.0f);
    const __half sh = __float2half_rn(scale);
    *scale_bits = __half_as_ushort(sh);
    const float eff = __half2float(sh);
    const float inv = (amax == 0.0f || eff == 0.0f) ? 0.0f : __frcp_rn(eff);
    int q[4];
#pragma unroll
    for (int j = 0; j < 4; j++) q[j] = round_away(__fmul_rn(v[j], inv));
    if (!plain)
#pragma unroll
      for (int j = 0; j < 4; j++) q[j] = max(-128, min(127, q[j]));
    codes = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  } else {
    int q[4];
    if (plain) {
      const float scale = quotient(amax, 7.0f, 1.0f / 7.0f), y = __frcp_rn(scale);
      *scale_bits = __half_as_ushort(__float2half_rn(scale));
#pragma unroll
      for (int j = 0; j < 4; j++) q[j] = round_away(quotient(v[j], scale, y));
    } else {
      const float scale = amax == 0.0f ? 1.0f : __fdiv_rn(amax, 7.0f);
      *scale_bits = __half_as_ushort(__float2half_rn(scale));
#pragma unroll
      for (int j = 0; j < 4; j++) q[j] = max(-8, min(7, round_away(__fdiv_rn(v[j], scale))));
    }
#pragma unroll
    for (int j = 0; j < 4; j++) codes += (uint32_t)(q[j] + 8) << (4 * j);
  }
  return codes;
}

// Lane i's part of a block at `dst` (2-byte aligned).
template <int DT>
__device__ __forceinline__ void store_block_part(uint8_t* dst, uint32_t i, uint32_t codes, uint16_t scale_bits) {
  uint16_t* d = reinterpret_cast<uint16_t*>(dst);
  if (i == 0) d[0] = scale_bits;
  if (DT == AION_CUDA_DTYPE_Q8_0) {
    d[1 + 2 * i] = (uint16_t)codes;
    d[2 + 2 * i] = (uint16_t)(codes >> 16);
  } else {
    d[1 + i] = (uint16_t)codes;
  }
}

// ---- append: a warp per piece of a new row, eight lanes per block ------------------------------------
// Four consecutive values as f32; VEC: the address is a multiple of their size.
template <bool VEC>
__device__ __forceinline__ void load_4(const float* p, float (&v)[4]) {
  if (VEC) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = p[j];
  }
}
template <bool VEC>
__device__ __forceinline__ void load_4(const __half* p, float (&v)[4]) {
  if (VEC) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&x.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = __half2float(p[j]);
  }
}

// A piece is 16 blocks of a row (four of each lane group): where the row goes is worked out once for them, and their
// loads are under way together.
constexpr int PIECE = 16;

template <int DT, typename T, bool VEC>
__global__ void __launch_bounds__(128) append_quantized_kernel(uint8_t* __restrict__ cache, const T* __restrict__ rows,
                                                               const int32_t* __restrict__ end_index, CacheGeom g, uint32_t new_len,
                                                               uint32_t blocks_per_row, uint32_t pieces_per_row, uint32_t pieces, int* fault) {
  constexpr int BB = DT == AION_CUDA_DTYPE_Q8_0 ? Q8_BYTES : Q4_BYTES;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const uint32_t lane = threadIdx.x & 31, i = lane & 7, warps = gridDim.x * (blockDim.x / 32);
  for (uint32_t piece = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; piece < pieces; piece += warps) {
    const uint32_t r = piece / pieces_per_row, first = (piece - r * pieces_per_row) * PIECE + lane / 8;
    const uint32_t b = r / new_len, t = r - b * new_len;
    float v[PIECE / 4][4];
#pragma unroll
    for (int k = 0; k < PIECE / 4; k++) {
      const uint32_t blk = first + 4 * k;
      if (blk < blocks_per_row) load_4<VEC>(rows + ((uint64_t)r * blocks_per_row + blk) * QK + 4 * i, v[k]);
      else v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.0f;
    }
    bool bad = false;
    const int64_t row = append_row(g, b, end_index[b], t, new_len, &bad);
    if (bad && lane == 0) atomicCAS(fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
    if (row < 0) continue;   // the same for the whole warp
    uint8_t* dst = cache + (uint64_t)row * blocks_per_row * BB;
#pragma unroll
    for (int k = 0; k < PIECE / 4; k++) {
      const uint32_t blk = first + 4 * k;
      uint16_t scale;
      const uint32_t codes = quantize_4<DT>(v[k], &scale);
      if (blk < blocks_per_row) store_block_part<DT>(dst + blk * BB, i, codes, scale);
    }
  }
}

// ---- read: values of logical steps -----------------------------------------------------------------
// The row that holds step start[b] + t, negative: none, and zeros are read.
__device__ __forceinline__ int64_t read_row(const CacheGeom& g, const int32_t* start, const int32_t* lengths, uint32_t b, uint32_t t, bool* bad) {
  const ReadSpan s = read_span(g, start, lengths, b);
  *bad = s.bad;
  const uint64_t step = (uint64_t)(start && !s.bad ? start[b] : 0) + t;
  if (step < s.lo || step >= s.hi) return -1;
  const int64_t row = cache_row(g, b, (uint32_t)step);
  *bad = row < 0;
  return row;
}

template <typename O>
__device__ __forceinline__ O as_out(float v) { return (O)v; }
template <>
__device__ __forceinline__ __half as_out<__half>(float v) { return __float2half_rn(v); }

// One value of a stored row: element e of a row at `p`.
template <int DT>
__device__ __forceinline__ float row_value(const uint8_t* p, uint32_t e) {
  if (DT == AION_CUDA_DTYPE_F32) return reinterpret_cast<const float*>(p)[e];
  if (DT == AION_CUDA_DTYPE_F16) return __half2float(reinterpret_cast<const __half*>(p)[e]);
  constexpr int BB = DT == AION_CUDA_DTYPE_Q8_0 ? Q8_BYTES : Q4_BYTES;
  const uint8_t* blk = p + (uint64_t)(e / QK) * BB;
  const uint32_t t = e % QK;
  const float scale = __half2float(*reinterpret_cast<const __half*>(blk));
  int q;
  if (DT == AION_CUDA_DTYPE_Q8_0) q = (int8_t)blk[2 + t];
  else q = (int)((blk[2 + (t >> 1)] >> (4 * (t & 1))) & 15) - 8;
  return __fmul_rn((float)q, scale);
}

// One thread per value: rows of any size at any address.
template <int DT, typename O>
__global__ void __launch_bounds__(256) sequence_read_kernel(O* __restrict__ out, const uint8_t* __restrict__ cache,
                                                            const int32_t* __restrict__ start, const int32_t* __restrict__ lengths,
                                                            CacheGeom g, uint32_t out_len, uint32_t row_values, uint64_t row_bytes,
                                                            uint64_t count, int* fault) {
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  for (uint64_t i = blockIdx.x * (uint64_t)blockDim.x + threadIdx.x; i < count; i += (uint64_t)gridDim.x * blockDim.x) {
    const uint64_t r = i / row_values;
    const uint32_t e = (uint32_t)(i - r * row_values);
    const uint32_t b = (uint32_t)(r / out_len), t = (uint32_t)(r - (uint64_t)b * out_len);
    bool bad;
    const int64_t row = read_row(g, start, lengths, b, t, &bad);
    const float v = row >= 0 ? row_value<DT>(cache + (uint64_t)row * row_bytes, e) : 0.0f;
    if (bad) atomicCAS(fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
    out[i] = as_out<O>(v);
  }
}

// Eight consecutive values of a stored row as f32; e is a multiple of 8, of rows that hold whole eights.
template <int DT>
struct Raw8 {
  uint32_t w[DT == AION_CUDA_DTYPE_F32 ? 8 : DT == AION_CUDA_DTYPE_F16 ? 4 : DT == AION_CUDA_DTYPE_Q8_0 ? 3 : 2];
  __device__ __forceinline__ void load(const uint8_t* row, uint32_t e) {
    if constexpr (DT == AION_CUDA_DTYPE_F32) {
      const uint4 a = *reinterpret_cast<const uint4*>(row + 4ull * e), b = *reinterpret_cast<const uint4*>(row + 4ull * e + 16);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    } else if constexpr (DT == AION_CUDA_DTYPE_F16) {
      const uint4 a = *reinterpret_cast<const uint4*>(row + 2ull * e);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
      // Blocks lie on 2-byte boundaries only.
      constexpr bool Q8 = DT == AION_CUDA_DTYPE_Q8_0;
      const uint16_t* blk = reinterpret_cast<const uint16_t*>(row + (uint64_t)(e / QK) * (Q8 ? Q8_BYTES : Q4_BYTES));
      const uint32_t j = e % QK / 8;
      w[0] = blk[0];
      if (Q8) {
        w[1] = blk[1 + 4 * j] | (uint32_t)blk[2 + 4 * j] << 16;
        w[2] = blk[3 + 4 * j] | (uint32_t)blk[4 + 4 * j] << 16;
      } else {
        w[1] = blk[1 + 2 * j] | (uint32_t)blk[2 + 2 * j] << 16;
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (uint32_t& x : w) x = 0;
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; k++) {
      if constexpr (DT == AION_CUDA_DTYPE_F32) v[k] = __uint_as_float(w[k]);
      else if constexpr (DT == AION_CUDA_DTYPE_F16) v[k] = __half2float(__ushort_as_half((unsigned short)(w[k / 2] >> (16 * (k & 1)))));
      else {
        const float scale = __half2float(__ushort_as_half((unsigned short)w[0]));
        int q;
        if constexpr (DT == AION_CUDA_DTYPE_Q8_0) q = (int)(w[1 + k / 4] << (24 - 8 * (k & 3))) >> 24;
        else q = (int)((w[1] >> (4 * k)) & 15) - 8;
        v[k] = __fmul_rn((float)q, scale);
      }
    }
  }
};
__device__ __forceinline__ void store_8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store_8(__half* p, const float (&v)[8]) {
  __half2 h[4];
#pragma unroll
  for (int k = 0; k < 4; k++) h[k] = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

// A warp per piece of a row, eight values per lane and step: where the row lies is worked out once for a piece, and
// the loads of its four steps are under way together.
constexpr int READ_STEPS = 4;

template <int DT, typename O>
__global__ void __launch_bounds__(128) sequence_read8_kernel(O* __restrict__ out, const uint8_t* __restrict__ cache,
                                                             const int32_t* __restrict__ start, const int32_t* __restrict__ lengths,
                                                             CacheGeom g, uint32_t out_len, uint32_t row_eights, uint64_t row_bytes,
                                                             uint32_t pieces_per_row, uint32_t pieces, int* fault) {
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const uint32_t lane = threadIdx.x & 31, warps = gridDim.x * (blockDim.x / 32);
  for (uint32_t piece = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; piece < pieces; piece += warps) {
    const uint32_t r = piece / pieces_per_row, first = (piece - r * pieces_per_row) * (32 * READ_STEPS) + lane;
    const uint32_t b = r / out_len, t = r - b * out_len;
    bool bad;
    const int64_t row = read_row(g, start, lengths, b, t, &bad);
    if (bad && lane == 0) atomicCAS(fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
    const uint8_t* src = cache + (uint64_t)(row < 0 ? 0 : row) * row_bytes;
    Raw8<DT> raw[READ_STEPS];
#pragma unroll
    for (int k = 0; k < READ_STEPS; k++) {
      raw[k].zero();
      if (row >= 0 && first + 32 * k < row_eights) raw[k].load(src, 8 * (first + 32 * k));
    }
#pragma unroll
    for (int k = 0; k < READ_STEPS; k++)
      if (first + 32 * k < row_eights) {
        float v[8];
        raw[k].values(v);
        // a row that is not held: zeros, not minus zeros (0 x -8)
        if (row < 0)
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] = 0.0f;
        store_8(out + ((uint64_t)r * row_eights + first + 32 * k) * 8, v);
      }
  }
}

// ---- norm, rotation and append of one projection row: one CTA per (request, new row) -------------
struct NormRopeParams {
  float* q_out;
  const float* qkv;
  const float *q_gamma, *k_gamma;
  const int32_t *positions, *end_index;
  uint8_t *k_cache, *v_cache;
  uint32_t len, h_q, h_kv, d;
  uint64_t ld;
  uint32_t rope_pairs;
  float step, scale_factor, eps;
  uint32_t k_dtype, v_dtype;
  CacheGeom geom;
  int* fault;
};

constexpr int NR_THREADS = 128;
constexpr int NR_WARPS = NR_THREADS / 32;

// One head, held in shared memory by one warp, into its cache row.
__device__ __forceinline__ void store_head(const float* x, uint32_t d, uint32_t dtype, uint8_t* cache, uint64_t head_index, int lane) {
  if (dtype == AION_CUDA_DTYPE_F16) {
    __half* dst = reinterpret_cast<__half*>(cache) + head_index * d;
    for (uint32_t c = lane; c < d; c += 32) dst[c] = __float2half_rn(x[c]);
    return;
  }
  const uint32_t blocks = d / QK, i = lane & 7;
  for (uint32_t k0 = 0; k0 < blocks; k0 += 4) {
    const uint32_t k = k0 + lane / 8;
    const bool on = k < blocks;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = on ? x[k * QK + 4 * i + j] : 0.0f;
    uint16_t scale;
    if (dtype == AION_CUDA_DTYPE_Q8_0) {
      const uint32_t codes = quantize_4<AION_CUDA_DTYPE_Q8_0>(v, &scale);
      if (on) store_block_part<AION_CUDA_DTYPE_Q8_0>(cache + (head_index * blocks + k) * Q8_BYTES, i, codes, scale);
    } else {
      const uint32_t codes = quantize_4<AION_CUDA_DTYPE_Q4_0>(v, &scale);
      if (on) store_block_part<AION_CUDA_DTYPE_Q4_0>(cache + (head_index * blocks + k) * Q4_BYTES, i, codes, scale);
    }
  }
}

__global__ void __launch_bounds__(NR_THREADS) qk_norm_rope_append_kernel(const NormRopeParams p) {
  extern __shared__ float nr_smem[];   // cos, sin of the row's angles; one head per warp
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const uint32_t half = p.d / 2;
  float* cs = nr_smem;
  float* sn = cs + half;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* x = sn + half + (uint32_t)warp * p.d;
  const uint64_t row = blockIdx.x;
  const uint32_t b = (uint32_t)(row / p.len), l = (uint32_t)(row - (uint64_t)b * p.len);
  bool bad;
  const int64_t dst = append_row(p.geom, b, p.end_index[b], l, p.len, &bad);
  if (bad && threadIdx.x == 0) atomicCAS(p.fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
  const float pos = (float)p.positions[row];
  for (uint32_t i = threadIdx.x; i < p.rope_pairs; i += NR_THREADS) {
    // Frequency of pair i by repeated f32 multiplies, as the RoPE step builds it.
    float f = p.scale_factor;
    for (uint32_t j = 0; j < i; j++) f *= p.step;
    double s, c;
    sincos((double)(pos * f), &s, &c);
    cs[i] = (float)c, sn[i] = (float)s;
  }
  __syncthreads();
  const float* src = p.qkv + row * p.ld;
  for (uint32_t h = warp; h < p.h_q + 2 * p.h_kv; h += NR_WARPS) {
    const float* xs = src + (uint64_t)h * p.d;
    const bool is_q = h < p.h_q, is_v = h >= p.h_q + p.h_kv;
    for (uint32_t c = lane; c < p.d; c += 32) x[c] = xs[c];
    __syncwarp();
    if (!is_v) {
      const float* gamma = is_q ? p.q_gamma : p.k_gamma;
      if (gamma) {
        // The sum of squares is taken in 64 bits (each square is exact there): its f32 root does not depend on
        // the order of the sum, so a code on a border does not either.
        double ss = 0.0;
        for (uint32_t c = lane; c < p.d; c += 32) ss += (double)x[c] * (double)x[c];
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
        const double ms = ss / (double)p.d + (double)p.eps;
        if (!(ms > 0.0) || isinf(ms)) {
          if (lane == 0) atomicCAS(p.fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
          continue;
        }
        const float inv = (float)(1.0 / sqrt(ms));
        for (uint32_t c = lane; c < p.d; c += 32) x[c] = (x[c] * inv) * gamma[c];
        __syncwarp();
      }
      for (uint32_t i = lane; i < p.rope_pairs; i += 32) {
        const float a = x[i], c = x[half + i];
        x[i] = a * cs[i] - c * sn[i];
        x[half + i] = a * sn[i] + c * cs[i];
      }
      __syncwarp();
    }
    if (is_q) {
      float* qo = p.q_out + (row * p.h_q + h) * p.d;
      for (uint32_t c = lane; c < p.d; c += 32) qo[c] = x[c];
    } else if (dst >= 0) {
      const uint32_t hk = is_v ? h - p.h_q - p.h_kv : h - p.h_q;
      store_head(x, p.d, is_v ? p.v_dtype : p.k_dtype, is_v ? p.v_cache : p.k_cache, (uint64_t)dst * p.h_kv + hk, lane);
    }
    __syncwarp();
  }
}

// The same for heads of 64, 128 and 256: D / 8 lanes hold a head, each of them the values 4j .. 4j + 3 of its first half
// and of its second half (the pairs that rotate together; eight lanes hold a block). The warps' loads of all rows, 256
// values each, are cut into equal runs, one per resident warp: a warp works out a row's angles, a few a lane, keeps them
// in registers while it walks the row's heads, and has the next load's values on their way.
constexpr int NRF_THREADS = 128;
constexpr int NRF_CTAS = 6;   // an SM: 80 registers a thread (5 CTAs, 6 and, with spills, 8: 139, 134 and 147 us for 16000 rows of 16 heads of 256)

// A lane's four values into a head: `dst` is where they belong in an f16 cache, or their block in a quantized one.
__device__ __forceinline__ void store_4(uint32_t dtype, uint8_t* dst, uint32_t i, const float (&v)[4], bool on) {
  if (dtype == AION_CUDA_DTYPE_F16) {
    const __half2 h[2] = {__floats2half2_rn(v[0], v[1]), __floats2half2_rn(v[2], v[3])};
    if (on) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(h);
    return;
  }
  uint16_t scale;
  if (dtype == AION_CUDA_DTYPE_Q8_0) {
    const uint32_t codes = quantize_4<AION_CUDA_DTYPE_Q8_0>(v, &scale);
    if (on) store_block_part<AION_CUDA_DTYPE_Q8_0>(dst, i, codes, scale);
  } else {
    const uint32_t codes = quantize_4<AION_CUDA_DTYPE_Q4_0>(v, &scale);
    if (on) store_block_part<AION_CUDA_DTYPE_Q4_0>(dst, i, codes, scale);
  }
}

// 1 / sqrt(x) of a double to the last bits of a float: the f32 estimate, two steps of Newton's iteration in f64.
__device__ __forceinline__ float inverse_root(double x) {
  if (!(x > 1e-30 && x < 1e30)) return (float)(1.0 / sqrt(x));
  double y = (double)rsqrtf((float)x);
  const double h = 0.5 * x;
  y = y * (1.5 - h * y * y);
  y = y * (1.5 - h * y * y);
  return (float)y;
}

template <int D>
__global__ void __launch_bounds__(NRF_THREADS, NRF_CTAS) qk_norm_rope_append_lanes_kernel(const NormRopeParams p, uint32_t total, uint32_t run) {
  constexpr int LPH = D / 8, HPW = 32 / LPH, HALF = D / 2, PPL = D / 64;   // lanes a head, heads a load, pairs a lane works out
  ptx::pdl_launch_dependents();
  const uint32_t lane = threadIdx.x & 31, j = lane % LPH;
  // Frequencies of this lane's pairs by repeated f32 multiplies, as the RoPE step builds them.
  float freq[PPL];
  freq[0] = p.scale_factor;
  for (uint32_t k = 0; k < lane * PPL; k++) freq[0] *= p.step;
#pragma unroll
  for (int k = 1; k < PPL; k++) freq[k] = freq[k - 1] * p.step;
  ptx::pdl_wait();
  const bool norms = p.q_gamma || p.k_gamma;
  // Bytes of a head in each cache, and where this lane's values of its first and second half lie in it.
  auto size_of = [](uint32_t dt, uint32_t values) {
    return dt == AION_CUDA_DTYPE_F16 ? values * 2 : values / QK * (dt == AION_CUDA_DTYPE_Q8_0 ? Q8_BYTES : Q4_BYTES);
  };
  const uint32_t k_head = size_of(p.k_dtype, D), k_at = size_of(p.k_dtype, 4 * j), v_head = size_of(p.v_dtype, D), v_at = size_of(p.v_dtype, 4 * j);
  const uint32_t slots = p.h_q + 2 * p.h_kv, loads = (slots + HPW - 1) / HPW;   // heads of a row, and the warp's loads of them
  const uint64_t begin = (uint64_t)run * (blockIdx.x * (NRF_THREADS / 32) + threadIdx.x / 32);
  if (begin >= total) return;
  uint32_t left = min(run, total - (uint32_t)begin), row = (uint32_t)begin / loads, n = (uint32_t)begin - row * loads;
  float4 ahead[2];
  auto load = [&](uint32_t r, uint32_t k) {
    const uint32_t h = min(k * HPW + lane / LPH, slots - 1);
    const float* src = p.qkv + (uint64_t)r * p.ld + h * D + 4 * j;
    ahead[0] = *reinterpret_cast<const float4*>(src);
    ahead[1] = *reinterpret_cast<const float4*>(src + HALF);
  };
  load(row, n);
  while (left > 0) {
    const uint32_t b = row / p.len, l = row - b * p.len;
    bool bad;
    const int64_t dst = append_row(p.geom, b, p.end_index[b], l, p.len, &bad);
    if (bad && lane == 0) atomicCAS(p.fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
    uint8_t* const k_row = p.k_cache + (uint64_t)(dst < 0 ? 0 : dst) * p.h_kv * k_head + k_at;
    uint8_t* const v_row = p.v_cache + (uint64_t)(dst < 0 ? 0 : dst) * p.h_kv * v_head + v_at;
    // the angles of pairs 4j .. 4j + 3
    float cs[4], sn[4];
    {
      const float pos = (float)p.positions[row];
      float c[PPL], s[PPL];
#pragma unroll
      for (int k = 0; k < PPL; k++) {
        c[k] = 1.0f, s[k] = 0.0f;
        if (lane * PPL + k < p.rope_pairs) {
          double sd, cd;
          sincos((double)(pos * freq[k]), &sd, &cd);
          c[k] = (float)cd, s[k] = (float)sd;
        }
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        cs[k] = PPL == 4 ? c[k % PPL] : __shfl_sync(FULL, c[k % PPL], (4 * j + k) / PPL);
        sn[k] = PPL == 4 ? s[k % PPL] : __shfl_sync(FULL, s[k % PPL], (4 * j + k) / PPL);
      }
    }
    for (; n < loads && left > 0; n++, left--) {
      float x[2][4] = {{ahead[0].x, ahead[0].y, ahead[0].z, ahead[0].w}, {ahead[1].x, ahead[1].y, ahead[1].z, ahead[1].w}};
      if (left > 1) load(n + 1 < loads ? row : row + 1, n + 1 < loads ? n + 1 : 0);
      const uint32_t h = n * HPW + lane / LPH;
      const bool on = h < slots, is_q = h < p.h_q, is_v = h >= p.h_q + p.h_kv;
      bool good = on;
      if (norms && n * HPW < p.h_q + p.h_kv) {   // (every lane takes part in the shuffles)
        // The sum of squares is taken in 64 bits (each square is exact there): its f32 root does not depend on
        // the order of the sum, so a code on a border does not either.
        double ss = 0.0;
#pragma unroll
        for (int k = 0; k < 8; k++) ss += (double)x[k >> 2][k & 3] * (double)x[k >> 2][k & 3];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
        if (!is_v && (is_q ? p.q_gamma : p.k_gamma)) {
          const double ms = ss * (1.0 / D) + (double)p.eps;   // D is a power of two
          if (!(ms > 0.0) || isinf(ms)) {
            if (on && j == 0) atomicCAS(p.fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
            good = false;
          }
          const float inv = inverse_root(ms);
          const float* gamma = (is_q ? p.q_gamma : p.k_gamma) + 4 * j;   // (a kilobyte that stays in L1)
#pragma unroll
          for (int k = 0; k < 8; k++) x[k >> 2][k & 3] = (x[k >> 2][k & 3] * inv) * __ldg(gamma + (k & 3) + (k >> 2) * HALF);
        }
      }
      if (!is_v) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float a = x[0][k], b2 = x[1][k];
          const bool turn = 4 * j + k < p.rope_pairs;
          x[0][k] = turn ? a * cs[k] - b2 * sn[k] : a;
          x[1][k] = turn ? a * sn[k] + b2 * cs[k] : b2;
        }
      }
      if (is_q && good) {
        float* qo = p.q_out + ((uint64_t)row * p.h_q + h) * D + 4 * j;
        *reinterpret_cast<float4*>(qo) = make_float4(x[0][0], x[0][1], x[0][2], x[0][3]);
        *reinterpret_cast<float4*>(qo + HALF) = make_float4(x[1][0], x[1][1], x[1][2], x[1][3]);
      }
      // All lanes go through the quantizer of each cache that the warp has heads for: its maxima are taken by shuffles.
      if ((n + 1) * HPW > p.h_q && n * HPW < p.h_q + p.h_kv) {
        const bool to_k = good && !is_q && !is_v && dst >= 0;
        uint8_t* at = k_row + (to_k ? h - p.h_q : 0) * k_head;
        store_4(p.k_dtype, at, j & 7, x[0], to_k);
        store_4(p.k_dtype, at + k_head / 2, j & 7, x[1], to_k);
      }
      if ((n + 1) * HPW > p.h_q + p.h_kv) {
        const bool to_v = on && is_v && dst >= 0;
        uint8_t* at = v_row + (to_v ? h - p.h_q - p.h_kv : 0) * v_head;
        store_4(p.v_dtype, at, j & 7, x[0], to_v);
        store_4(p.v_dtype, at + v_head / 2, j & 7, x[1], to_v);
      }
    }
    row++, n = 0;
  }
}

// ---- host side ---------------------------------------------------------------------------------------
bool quantized(uint32_t dt) { return dt == AION_CUDA_DTYPE_Q8_0 || dt == AION_CUDA_DTYPE_Q4_0; }

// Bytes of `values` consecutive values of a cache (whole blocks where it is quantized).
uint64_t cache_bytes(uint32_t dt, uint64_t values) {
  return quantized(dt) ? values / QK * block_bytes_of(dt) : values * (dt == AION_CUDA_DTYPE_F32 ? 4 : 2);
}

// The geometry of a cache and the number of its rows.
int32_t cache_geom(uint64_t batch, uint64_t t_cap, uint32_t rolling, const AionCudaOperand& table, uint64_t page_tokens, uint64_t pool_pages,
                   const char* what, CacheGeom* g, uint64_t* rows) {
  if (t_cap == 0) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: empty cache", what);
  if (t_cap > 0x7FFFFFFFull || batch > 0x7FFFFFFFull) return fail(AION_CUDA_UNSUPPORTED, "%s: a cache of more than 2^31 - 1 steps or requests", what);
  *g = CacheGeom{};
  g->t_cap = (uint32_t)t_cap;
  g->rolling = rolling ? 1u : 0u;
  *rows = batch * t_cap;
  if (table.handle) {
    if (rolling) return fail(AION_CUDA_UNSUPPORTED, "%s: a rolling cache cannot be paged", what);
    if (page_tokens == 0 || pool_pages == 0) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: page_tokens and pool_pages must be positive", what);
    if (page_tokens > 0x7FFFFFFFull || pool_pages > 0x7FFFFFFFull) return fail(AION_CUDA_UNSUPPORTED, "%s: pool beyond what the kernels index", what);
    g->page_tokens = (uint32_t)page_tokens;
    g->pool_pages = (uint32_t)pool_pages;
    g->pages_per_request = (uint32_t)((t_cap + page_tokens - 1) / page_tokens);
    *rows = pool_pages * page_tokens;
    if (int32_t st = resolve(table, batch * g->pages_per_request * sizeof(int32_t), what, &g->table)) return st;
  }
  return AION_CUDA_OK;
}

// A stretch of device memory that a step reads or writes; p null: an operand that is absent.
struct Span {
  const void* p;
  uint64_t bytes;
};
// What one warp writes no other may read or write: no written operand overlaps another one, read or written.
int32_t check_apart(const char* what, std::initializer_list<Span> written, std::initializer_list<Span> read) {
  auto overlap = [](const Span& a, const Span& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return a.p && b.p && x < y + b.bytes && y < x + a.bytes;
  };
  for (const Span& w : written) {
    for (const Span& o : written)
      if (&o != &w && overlap(w, o)) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: operands overlap", what);
    for (const Span& o : read)
      if (overlap(w, o)) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: operands overlap", what);
  }
  return AION_CUDA_OK;
}

unsigned blocks_for(const AionCudaDevice* dev, uint64_t items, unsigned per_block) {
  const uint64_t want = ceil_div(items, (uint64_t)per_block), cap = (uint64_t)dev->sm_count * 16;
  return (unsigned)(want < cap ? want : cap);
}

template <int DT, typename T>
int32_t launch_append_as(AionCudaDevice* dev, const AionCudaSequenceAppend* s, uint8_t* cache, const T* rows, const int32_t* idx, const CacheGeom& g) {
  const uint64_t bpr = s->heads * s->head_dim / QK, ppr = ceil_div(bpr, (uint64_t)PIECE), pieces = s->batch * s->new_len * ppr;
  if (pieces > 0x7FFFFFFFull) return fail(AION_CUDA_UNSUPPORTED, "sequence_append: too many rows for one launch");
  const bool vec = (reinterpret_cast<uintptr_t>(rows) & (4 * sizeof(T) - 1)) == 0;
  AION_CUDA_TRY(launch_pdl(vec ? append_quantized_kernel<DT, T, true> : append_quantized_kernel<DT, T, false>, dim3(blocks_for(dev, pieces, 4)), dim3(128), 0,
                           dev->stream, cache, rows, idx, g, (uint32_t)s->new_len, (uint32_t)bpr, (uint32_t)ppr, (uint32_t)pieces, dev->fault_dev));
  return AION_CUDA_OK;
}

template <typename T>
int32_t launch_append(AionCudaDevice* dev, const AionCudaSequenceAppend* s, uint8_t* cache, const T* rows, const int32_t* idx, const CacheGeom& g) {
  if (s->dtype == AION_CUDA_DTYPE_Q8_0) return launch_append_as<AION_CUDA_DTYPE_Q8_0, T>(dev, s, cache, rows, idx, g);
  return launch_append_as<AION_CUDA_DTYPE_Q4_0, T>(dev, s, cache, rows, idx, g);
}

template <int DT, typename O>
int32_t launch_read_as(AionCudaDevice* dev, const AionCudaSequenceRead* s, O* out, const uint8_t* cache, const int32_t* start, const int32_t* lengths,
                       const CacheGeom& g) {
  const uint64_t row_values = s->heads * s->head_dim, count = s->batch * s->out_len * row_values;
  const uint64_t row_bytes = cache_bytes(s->dtype, row_values);
  // Eight values at a time where rows are whole eights on 16-byte boundaries (of a quantized cache: of out alone).
  const uint64_t ppr = ceil_div(row_values / 8, (uint64_t)(32 * READ_STEPS)), pieces = s->batch * s->out_len * ppr;
  const uintptr_t addr = reinterpret_cast<uintptr_t>(out) | (quantized(s->dtype) ? 0 : reinterpret_cast<uintptr_t>(cache) | row_bytes);
  if (row_values % 8 == 0 && (addr & 15) == 0 && pieces <= 0x7FFFFFFFull) {
    AION_CUDA_TRY(launch_pdl(sequence_read8_kernel<DT, O>, dim3(blocks_for(dev, pieces, 4)), dim3(128), 0, dev->stream, out, cache, start, lengths, g,
                             (uint32_t)s->out_len, (uint32_t)(row_values / 8), row_bytes, (uint32_t)ppr, (uint32_t)pieces, dev->fault_dev));
  } else {
    AION_CUDA_TRY(launch_pdl(sequence_read_kernel<DT, O>, dim3(blocks_for(dev, count, 256)), dim3(256), 0, dev->stream, out, cache, start, lengths, g,
                             (uint32_t)s->out_len, (uint32_t)row_values, row_bytes, count, dev->fault_dev));
  }
  return AION_CUDA_OK;
}

template <typename O>
int32_t launch_read(AionCudaDevice* dev, const AionCudaSequenceRead* s, O* out, const uint8_t* cache, const int32_t* start, const int32_t* lengths,
                    const CacheGeom& g) {
  switch (s->dtype) {
    case AION_CUDA_DTYPE_F32: return launch_read_as<AION_CUDA_DTYPE_F32>(dev, s, out, cache, start, lengths, g);
    case AION_CUDA_DTYPE_F16: return launch_read_as<AION_CUDA_DTYPE_F16>(dev, s, out, cache, start, lengths, g);
    case AION_CUDA_DTYPE_Q8_0: return launch_read_as<AION_CUDA_DTYPE_Q8_0>(dev, s, out, cache, start, lengths, g);
    default: return launch_read_as<AION_CUDA_DTYPE_Q4_0>(dev, s, out, cache, start, lengths, g);
  }
}

}  // namespace

int32_t append_quantized(AionCudaDevice* dev, const AionCudaSequenceAppend* s) {
  const char* what = "sequence_append";
  if (s->new_dtype != AION_CUDA_DTYPE_F32 && s->new_dtype != AION_CUDA_DTYPE_F16)
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: new_kv dtype %u", what, s->new_dtype);
  if (s->batch == 0 || s->new_len == 0 || s->heads == 0 || s->head_dim == 0) return AION_CUDA_OK;
  if (s->head_dim % QK) return fail(AION_CUDA_UNSUPPORTED, "%s: a quantized cache needs heads of whole 32-blocks, got %llu", what, (unsigned long long)s->head_dim);
  if (s->heads > (1u << 16) || s->head_dim > (1u << 16)) return fail(AION_CUDA_UNSUPPORTED, "%s: head geometry", what);
  if (s->new_len > 0x7FFFFFFFull) return fail(AION_CUDA_UNSUPPORTED, "%s: too many rows for one launch", what);
  CacheGeom g;
  uint64_t rows;
  if (int32_t st = cache_geom(s->batch, s->t_cap, s->rolling, s->page_table, s->page_tokens, s->pool_pages, what, &g, &rows)) return st;
  const uint64_t row_values = s->heads * s->head_dim;
  if (rows > (1ull << 40) / row_values * 64 || s->batch * s->new_len > (1ull << 31)) return fail(AION_CUDA_UNSUPPORTED, "%s: shape beyond what the kernels index", what);
  uint8_t *cache, *nk;
  const int32_t* idx;
  if (int32_t st = resolve(s->cache, cache_bytes(s->dtype, rows * row_values), "sequence_append.cache", &cache)) return st;
  const uint64_t eb = s->new_dtype == AION_CUDA_DTYPE_F32 ? 4 : 2;
  if (int32_t st = resolve(s->new_kv, s->batch * s->new_len * row_values * eb, "sequence_append.new_kv", &nk)) return st;
  if (int32_t st = resolve(s->end_index, s->batch * sizeof(int32_t), "sequence_append.end_index", &idx)) return st;
  if ((reinterpret_cast<uintptr_t>(cache) & 1) || (reinterpret_cast<uintptr_t>(nk) & (eb - 1)))
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: misaligned operand", what);
  if (int32_t st = check_apart(what, {{cache, cache_bytes(s->dtype, rows * row_values)}},
                               {{nk, s->batch * s->new_len * row_values * eb}, {idx, s->batch * sizeof(int32_t)}, {g.table, s->batch * g.pages_per_request * sizeof(int32_t)}}))
    return st;
  if (int32_t st = dev->make_current()) return st;
  if (eb == 4) return launch_append(dev, s, cache, reinterpret_cast<const float*>(nk), idx, g);
  return launch_append(dev, s, cache, reinterpret_cast<const __half*>(nk), idx, g);
}

}  // namespace aion

using namespace aion;

extern "C" {

int32_t aion_cuda_sequence_read(AionCudaDevice* dev, const AionCudaSequenceRead* s) {
  const char* what = "sequence_read";
  if (!dev || !s) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: null argument", what);
  if (!quantized(s->dtype) && s->dtype != AION_CUDA_DTYPE_F16 && s->dtype != AION_CUDA_DTYPE_F32)
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: cache dtype %u", what, s->dtype);
  if (s->out_dtype != AION_CUDA_DTYPE_F16 && s->out_dtype != AION_CUDA_DTYPE_F32)
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: out dtype %u", what, s->out_dtype);
  if (s->batch == 0 || s->out_len == 0 || s->heads == 0 || s->head_dim == 0) return AION_CUDA_OK;
  if (quantized(s->dtype) && s->head_dim % QK)
    return fail(AION_CUDA_UNSUPPORTED, "%s: a quantized cache needs heads of whole 32-blocks, got %llu", what, (unsigned long long)s->head_dim);
  if (s->heads > (1u << 16) || s->head_dim > (1u << 16)) return fail(AION_CUDA_UNSUPPORTED, "%s: head geometry", what);
  if (s->out_len > 0x7FFFFFFFull) return fail(AION_CUDA_UNSUPPORTED, "%s: too many rows for one launch", what);
  CacheGeom g;
  uint64_t rows;
  if (int32_t st = cache_geom(s->batch, s->t_cap, s->rolling, s->page_table, s->page_tokens, s->pool_pages, what, &g, &rows)) return st;
  const uint64_t row_values = s->heads * s->head_dim;
  if (rows > (1ull << 40) / row_values * 64 || s->batch * s->out_len > (1ull << 31)) return fail(AION_CUDA_UNSUPPORTED, "%s: shape beyond what the kernels index", what);
  uint8_t *out, *cache;
  const int32_t *start = nullptr, *lengths = nullptr;
  const uint64_t ob = s->out_dtype == AION_CUDA_DTYPE_F32 ? 4 : 2;
  if (int32_t st = resolve(s->out, s->batch * s->out_len * row_values * ob, "sequence_read.out", &out)) return st;
  if (int32_t st = resolve(s->cache, cache_bytes(s->dtype, rows * row_values), "sequence_read.cache", &cache)) return st;
  if (s->start_index.handle)
    if (int32_t st = resolve(s->start_index, s->batch * sizeof(int32_t), "sequence_read.start_index", &start)) return st;
  if (s->lengths.handle)
    if (int32_t st = resolve(s->lengths, s->batch * sizeof(int32_t), "sequence_read.lengths", &lengths)) return st;
  const uintptr_t cache_align = s->dtype == AION_CUDA_DTYPE_F32 ? 3 : 1;
  if ((reinterpret_cast<uintptr_t>(cache) & cache_align) || (reinterpret_cast<uintptr_t>(out) & (ob - 1)))
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: misaligned operand", what);
  const uint64_t per_request = s->batch * sizeof(int32_t);
  if (int32_t st = check_apart(what, {{out, s->batch * s->out_len * row_values * ob}},
                               {{cache, cache_bytes(s->dtype, rows * row_values)}, {start, per_request}, {lengths, per_request}, {g.table, per_request * g.pages_per_request}}))
    return st;
  if (int32_t st = dev->make_current()) return st;
  if (ob == 4) return launch_read(dev, s, reinterpret_cast<float*>(out), cache, start, lengths, g);
  return launch_read(dev, s, reinterpret_cast<__half*>(out), cache, start, lengths, g);
}

int32_t aion_cuda_qk_norm_rope_append(AionCudaDevice* dev, const AionCudaQKNormRopeAppend* s) {
  const char* what = "qk_norm_rope_append";
  if (!dev || !s) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: null argument", what);
  for (uint32_t dt : {s->k_dtype, s->v_dtype})
    if (!quantized(dt) && dt != AION_CUDA_DTYPE_F16) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: cache dtype %u", what, dt);
  if ((s->q_gamma.handle || s->k_gamma.handle) && (!(s->eps > 0.0f) || !std::isfinite(s->eps)))
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: eps must be finite and > 0", what);
  if (s->head_dim == 0 || s->head_dim % 2 || s->head_dim > 1024 || s->h_q > (1u << 16) || s->h_kv > (1u << 16))
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: head geometry", what);
  if ((quantized(s->k_dtype) || quantized(s->v_dtype)) && s->head_dim % QK)
    return fail(AION_CUDA_UNSUPPORTED, "%s: a quantized cache needs heads of whole 32-blocks, got %llu", what, (unsigned long long)s->head_dim);
  if (s->batch == 0 || s->len == 0 || s->h_q + s->h_kv == 0) return AION_CUDA_OK;
  const uint64_t d = s->head_dim, width = (s->h_q + 2 * s->h_kv) * d, ld = s->ld_qkv ? s->ld_qkv : width;
  if (ld < width) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: ld_qkv is shorter than q | k | v", what);
  if (ld > (1ull << 32)) return fail(AION_CUDA_UNSUPPORTED, "%s: ld_qkv", what);
  if (s->len > 0x7FFFFFFFull || s->batch > 0x7FFFFFFFull || s->batch * s->len > 0x7FFFFFFFull)
    return fail(AION_CUDA_UNSUPPORTED, "%s: too many rows for one launch", what);
  // src/aion/backend/cpu/exec/rope.zig:43-50
  const float pf = std::floor(s->proportion * (float)(d / 2));
  if (!(pf >= 0.0f)) return fail(AION_CUDA_INVALID_ARGUMENT, "%s: proportion %g", what, (double)s->proportion);
  NormRopeParams p{};
  uint64_t cache_rows;
  if (int32_t st = cache_geom(s->batch, s->t_cap, s->rolling, s->page_table, s->page_tokens, s->pool_pages, what, &p.geom, &cache_rows)) return st;
  const uint64_t row_values = s->h_kv * d, rows = s->batch * s->len;
  if (row_values && cache_rows > (1ull << 40) / row_values * 64) return fail(AION_CUDA_UNSUPPORTED, "%s: shape beyond what the kernels index", what);
  if (s->h_q)
    if (int32_t st = resolve(s->q_out, rows * s->h_q * d * sizeof(float), "qk_norm_rope_append.q_out", &p.q_out)) return st;
  if (int32_t st = resolve(s->qkv, ((rows - 1) * ld + width) * sizeof(float), "qk_norm_rope_append.qkv", &p.qkv)) return st;
  if (s->q_gamma.handle)
    if (int32_t st = resolve(s->q_gamma, d * sizeof(float), "qk_norm_rope_append.q_gamma", &p.q_gamma)) return st;
  if (s->k_gamma.handle)
    if (int32_t st = resolve(s->k_gamma, d * sizeof(float), "qk_norm_rope_append.k_gamma", &p.k_gamma)) return st;
  if (int32_t st = resolve(s->positions, rows * sizeof(int32_t), "qk_norm_rope_append.positions", &p.positions)) return st;
  if (int32_t st = resolve(s->end_index, s->batch * sizeof(int32_t), "qk_norm_rope_append.end_index", &p.end_index)) return st;
  if (s->h_kv) {
    if (int32_t st = resolve(s->k_cache, cache_bytes(s->k_dtype, cache_rows * row_values), "qk_norm_rope_append.k_cache", &p.k_cache)) return st;
    if (int32_t st = resolve(s->v_cache, cache_bytes(s->v_dtype, cache_rows * row_values), "qk_norm_rope_append.v_cache", &p.v_cache)) return st;
  }
  const uintptr_t f32s = reinterpret_cast<uintptr_t>(p.q_out) | reinterpret_cast<uintptr_t>(p.qkv) | reinterpret_cast<uintptr_t>(p.q_gamma) |
                         reinterpret_cast<uintptr_t>(p.k_gamma);
  if ((f32s & 3) || ((reinterpret_cast<uintptr_t>(p.k_cache) | reinterpret_cast<uintptr_t>(p.v_cache)) & 1))
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: misaligned operand", what);
  if (int32_t st = check_apart(what,
                               {{p.k_cache, cache_bytes(s->k_dtype, cache_rows * row_values)}, {p.v_cache, cache_bytes(s->v_dtype, cache_rows * row_values)},
                                {p.q_out, rows * s->h_q * d * sizeof(float)}},
                               {{p.qkv, ((rows - 1) * ld + width) * sizeof(float)}, {p.q_gamma, d * sizeof(float)}, {p.k_gamma, d * sizeof(float)},
                                {p.positions, rows * sizeof(int32_t)}, {p.end_index, s->batch * sizeof(int32_t)},
                                {p.geom.table, s->batch * p.geom.pages_per_request * sizeof(int32_t)}}))
    return st;
  if (int32_t st = dev->make_current()) return st;
  p.len = (uint32_t)s->len, p.h_q = (uint32_t)s->h_q, p.h_kv = (uint32_t)s->h_kv, p.d = (uint32_t)d;
  p.ld = ld;
  p.rope_pairs = pf > (float)(d / 2) ? (uint32_t)(d / 2) : (uint32_t)pf;
  p.step = (float)std::pow((double)s->base_frequency, (double)(-2.0f / (float)d));
  p.scale_factor = s->scale_factor, p.eps = s->eps;
  p.k_dtype = s->k_dtype, p.v_dtype = s->v_dtype;
  p.fault = dev->fault_dev;
  // Heads of 64, 128 and 256 at addresses of 16 bytes (8 in an f16 cache): eight values a lane.
  uintptr_t at16 = reinterpret_cast<uintptr_t>(p.q_out) | reinterpret_cast<uintptr_t>(p.qkv) | (ld * 4), at8 = 0;
  if (s->k_dtype == AION_CUDA_DTYPE_F16) at8 |= reinterpret_cast<uintptr_t>(p.k_cache);
  if (s->v_dtype == AION_CUDA_DTYPE_F16) at8 |= reinterpret_cast<uintptr_t>(p.v_cache);
  if ((d == 64 || d == 128 || d == 256) && (at16 & 15) == 0 && (at8 & 7) == 0) {
    const uint64_t total = rows * ceil_div(s->h_q + 2 * s->h_kv, 256 / d), resident = (uint64_t)dev->sm_count * NRF_CTAS * (NRF_THREADS / 32);
    const uint64_t run = ceil_div(total, resident);
    if (total <= 0x7FFFFFFFull) {
      const dim3 grid((unsigned)ceil_div(ceil_div(total, run), (uint64_t)(NRF_THREADS / 32))), block(NRF_THREADS);
#define AION_NRF(DD) AION_CUDA_TRY(launch_pdl(qk_norm_rope_append_lanes_kernel<DD>, grid, block, 0, dev->stream, p, (uint32_t)total, (uint32_t)run))
      if (d == 64) AION_NRF(64);
      else if (d == 128) AION_NRF(128);
      else AION_NRF(256);
#undef AION_NRF
      return AION_CUDA_OK;
    }
  }
  const size_t smem = (d + NR_WARPS * d) * sizeof(float);
  AION_CUDA_TRY(launch_pdl(qk_norm_rope_append_kernel, dim3((unsigned)rows), dim3(NR_THREADS), smem, dev->stream, p));
  return AION_CUDA_OK;
}

}  // extern "C"
