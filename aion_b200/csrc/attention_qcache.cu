// `Attention` over a quantized KV cache: K and V are q8_0 / q4_0 blocks of 32 along the head dimension, kept
// contiguous, as a ring, or in pages.
//
// With k_t = c_t * s_t (integer codes times the block's f16 scale), for every query row
//   logit_t = scale * sum_blocks s_t[block] * (q[block] . c_t[block])      (optional soft cap)
//   out[block] = sum_t softmax_t * s_t[block] * c_t[block]
// over the keys [lo, hi) of the row's window; zeros for an empty range. The codes are exact in any float type
// and the scales in f32, so only the f32 sums round: the result is f32 attention over the dequantized cache.
#include "attention_device.cuh"
#include "cache_geom.cuh"

namespace aion {

namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;

__device__ __forceinline__ CacheGeom geom_of(const AttnParams& p) {
  return CacheGeom{p.page_table, p.T, p.page_tokens, p.pages_per_request, p.pool_pages, p.rolling};
}

template <bool Q8>
__device__ __forceinline__ float block_value(const uint8_t* row, uint32_t e) {
  const uint8_t* blk = row + (uint64_t)(e >> 5) * (Q8 ? Q8_BYTES : Q4_BYTES);
  const uint32_t i = e & 31;
  const float scale = __half2float(*reinterpret_cast<const __half*>(blk));
  const int c = Q8 ? (int)(int8_t)blk[2 + i] : (int)((blk[2 + (i >> 1)] >> (4 * (i & 1))) & 15) - 8;
  return (float)c * scale;
}

// ------------------------------------------------------------------------------------
// any head size that is a multiple of 32: one CTA per output row (b, l, hq), 4 warps stride the keys, lanes
// stride the head dimension; per-warp online softmax, merged in shared memory.
// ------------------------------------------------------------------------------------
constexpr int ROW_WARPS = 4;
constexpr int MAX_DV_PER_LANE = 32;  // Dv <= 1024

template <bool KQ8, bool VQ8>
__global__ void __launch_bounds__(ROW_WARPS * 32) attn_qcache_row_kernel(const AttnParams p) {
  extern __shared__ float gsm[];  // q[Dk], then per warp: acc[Dv], m, l
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t row = blockIdx.x;
  const uint32_t hq = row % p.Hq;
  const uint32_t l = (row / p.Hq) % p.L;
  const uint32_t b = row / (p.Hq * p.L);
  const uint32_t hkv = hq / (p.Hq / p.Hkv);
  float* qs = gsm;
  float* wbuf = gsm + p.Dk + (size_t)warp * (p.Dv + 2);
  const uint64_t k_head = p.Dk / QK * (KQ8 ? Q8_BYTES : Q4_BYTES), v_head = p.Dv / QK * (VQ8 ? Q8_BYTES : Q4_BYTES);

  const CacheGeom geom = geom_of(p);
  const KeyRange kr = key_range(p, b, l);
  if (kr.bad && tid == 0) atomicExch(p.fault, FAULT_INVALID_ARGUMENT);
  for (uint32_t i = tid; i < p.Dk; i += blockDim.x) {
    const uint64_t at = (uint64_t)row * p.Dk + i;
    qs[i] = p.q_dtype == AION_CUDA_DTYPE_F32 ? static_cast<const float*>(p.q)[at] : __half2float(static_cast<const __half*>(p.q)[at]);
  }
  __syncthreads();

  float m_run = -INFINITY, l_run = 0.0f;
  float acc[MAX_DV_PER_LANE];
#pragma unroll
  for (int i = 0; i < MAX_DV_PER_LANE; i++) acc[i] = 0.0f;
  for (uint32_t t = kr.lo + warp; t < kr.hi; t += ROW_WARPS) {
    const int64_t kvr = cache_row(geom, b, t);
    if (kvr < 0) {
      if (lane == 0) atomicExch(p.fault, FAULT_INVALID_ARGUMENT);
      continue;
    }
    const uint8_t* krow = static_cast<const uint8_t*>(p.k) + ((uint64_t)kvr * p.Hkv + hkv) * k_head;
    const uint8_t* vrow = static_cast<const uint8_t*>(p.v) + ((uint64_t)kvr * p.Hkv + hkv) * v_head;
    float dot = 0.0f;
    for (uint32_t i = lane; i < p.Dk; i += 32) dot = fmaf(qs[i], block_value<KQ8>(krow, i), dot);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(FULL, dot, o);
    const float lg = soft_cap_logit(dot * p.scale, p.soft_cap) * LOG2E;
    const float m_new = fmaxf(m_run, lg);
    const float alpha = exp2f(m_run - m_new);
    const float pr = exp2f(lg - m_new);
    l_run = l_run * alpha + pr;
    m_run = m_new;
#pragma unroll
    for (int i = 0; i < MAX_DV_PER_LANE; i++) {
      const uint32_t d = lane + 32 * i;
      if (d < p.Dv) acc[i] = acc[i] * alpha + pr * block_value<VQ8>(vrow, d);
    }
  }
#pragma unroll
  for (int i = 0; i < MAX_DV_PER_LANE; i++) {
    const uint32_t d = lane + 32 * i;
    if (d < p.Dv) wbuf[d] = acc[i];
  }
  if (lane == 0) {
    wbuf[p.Dv] = m_run;
    wbuf[p.Dv + 1] = l_run;
  }
  __syncthreads();
  float* orow = p.out + (uint64_t)row * p.Dv;
  const float* base = gsm + p.Dk;
  float M = -INFINITY;
  for (int w = 0; w < ROW_WARPS; w++) M = fmaxf(M, base[(size_t)w * (p.Dv + 2) + p.Dv]);
  float lsum = 0.0f;
  for (int w = 0; w < ROW_WARPS; w++) {
    const float mw = base[(size_t)w * (p.Dv + 2) + p.Dv];
    lsum += (mw == -INFINITY) ? 0.0f : base[(size_t)w * (p.Dv + 2) + p.Dv + 1] * exp2f(mw - M);
  }
  const bool good = lsum > 0.0f && isfinite(lsum);
  if (!good && kr.hi > kr.lo && !kr.bad && tid == 0) atomicCAS(p.fault, FAULT_NONE, FAULT_NONFINITE);
  for (uint32_t d = tid; d < p.Dv; d += blockDim.x) {
    float o = 0.0f;
    for (int w = 0; w < ROW_WARPS; w++) {
      const float mw = base[(size_t)w * (p.Dv + 2) + p.Dv];
      if (mw != -INFINITY) o += base[(size_t)w * (p.Dv + 2) + d] * exp2f(mw - M);
    }
    orow[d] = good ? o / lsum : 0.0f;
  }
}

template <bool KQ8, bool VQ8>
int32_t launch_rows(AionCudaDevice* dev, const AttnParams& p) {
  const size_t smem = (p.Dk + ROW_WARPS * (p.Dv + 2)) * sizeof(float);
  attn_qcache_row_kernel<KQ8, VQ8><<<p.B * p.L * p.Hq, ROW_WARPS * 32, smem, dev->stream>>>(p);
  AION_CUDA_TRY(cudaGetLastError());
  return AION_CUDA_OK;
}

}  // namespace

int32_t attention_qcache_launch(AionCudaDevice* dev, AttnParams& p) {
  const bool kq8 = p.k_dtype == AION_CUDA_DTYPE_Q8_0, vq8 = p.v_dtype == AION_CUDA_DTYPE_Q8_0;
  if (p.image) return fail(AION_CUDA_UNSUPPORTED, "attention: no output image over a quantized cache");
  if (p.Dv > 32 * MAX_DV_PER_LANE || (p.Dk + ROW_WARPS * (p.Dv + 2)) * sizeof(float) > 48 * 1024)
    return fail(AION_CUDA_UNSUPPORTED, "attention: head dimensions %u / %u exceed the any-shape kernel", p.Dk, p.Dv);
  p.splits = 1;
  if (kq8) return vq8 ? launch_rows<true, true>(dev, p) : launch_rows<true, false>(dev, p);
  return vq8 ? launch_rows<false, true>(dev, p) : launch_rows<false, false>(dev, p);
}

}  // namespace aion
