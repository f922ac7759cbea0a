// What the attention kernels share: the step's parameters, the key range of a query row, the f16 tensor-core
// step and the last step of an output column.
#pragma once

#include <cfloat>
#include <cmath>

#include "act_image.cuh"
#include "common.cuh"
#include "ptx.cuh"

namespace aion {

constexpr float LOG2E = 1.4426950408889634f;

struct AttnParams {
  const void* q;
  const void* k;
  const void* v;
  float* out;
  const int32_t* positions;
  const int32_t* lengths;
  uint32_t B, L, Hq, Hkv, Dk, Dv, T;
  uint32_t q_dtype, k_dtype, v_dtype;
  uint32_t rolling;
  uint32_t win_left, win_right, win_chunk;
  float scale, soft_cap;
  uint32_t splits;
  uint32_t head_groups;  // ceil((Hq/Hkv) / 8)
  uint32_t col_heads;    // query heads of a head group: min(Hq/Hkv, 8)
  uint32_t pos_per_tile; // query positions sharing one 8-column MMA tile
  uint32_t l_blocks;     // blocks of positions per request
  const int32_t* page_table;  // [B][pages_per_request] page numbers, or null: K / V are [B, T, ...]
  uint32_t page_tokens, pages_per_request, pool_pages;
  float* partial;        // [unit][split][columns][Dv + 4]: sums, max, sum of weights, pad
  int* tickets;          // [unit]
  int* fault;
  // Optional: the quantized image of `out` as [B*L, Hq*Dv] rows (act_image.cuh), for the matmul
  // that consumes the attention output.
  uint8_t* image;
  ActImageLayout image_layout;
  uint32_t image_dtype;
  uint32_t wait_limit;   // polls a barrier wait makes before it gives up and reports FAULT_WAIT_EXPIRED
  uint32_t drop_first;   // test hook: every CTA leaves out the copies of its first stage, so that wait runs out
};

struct KeyRange {
  uint32_t lo, hi;
  bool bad;
};

// Window and ring clipping of one query row; flags inputs the reference rejects.
__device__ __forceinline__ KeyRange key_range(const AttnParams& p, uint32_t b, uint32_t l) {
  KeyRange r{0, 0, false};
  int64_t valid_end = p.T;
  if (p.lengths) {
    const int32_t e = p.lengths[b];
    if (e < 0) { r.bad = true; return r; }
    valid_end = e;
  }
  if (!p.rolling && valid_end > (int64_t)p.T) { r.bad = true; return r; }
  int64_t q_pos = l;
  if (p.positions) {
    const int32_t qp = p.positions[(uint64_t)b * p.L + l];
    if (qp < 0) { r.bad = true; return r; }
    q_pos = qp;
  }
  const int64_t anchor = p.win_chunk > 0 ? (q_pos / p.win_chunk) * p.win_chunk : q_pos;
  const int64_t span = p.win_chunk > 0 ? p.win_chunk : 1;
  int64_t lo = anchor - min(anchor, (int64_t)p.win_left);
  int64_t hi = min(valid_end, anchor + span + (int64_t)p.win_right);
  if (p.rolling && valid_end > (int64_t)p.T) lo = max(lo, valid_end - (int64_t)p.T);
  if (hi > lo) {
    r.lo = (uint32_t)lo;
    r.hi = (uint32_t)hi;
  }
  return r;
}

__device__ __forceinline__ float soft_cap_logit(float x, float cap) { return cap > 0.0f ? cap * tanhf(x / cap) : x; }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// K / V in q8_0 / q4_0 blocks (attention_qcache.cu).
int32_t attention_qcache_launch(AionCudaDevice* dev, AttnParams& p, uint32_t flags);

constexpr uint32_t NO_ROW = 0xFFFFFFFFu;

// The last step of one float4 of an output column: o / lsum (zeros for a column without keys), the store, and
// the quantized image of the output. All 32 lanes of a warp call it together (a column that does not exist
// passes on = false). Callers run it in a loop that is NOT unrolled: this code runs once per CTA, at the very
// end, on the CTA every other one is waiting for, and run once it costs what fetching its instructions costs
// (four columns spelled out side by side took 4 to 5 us, most of it in the quantizer).
template <int D>
__device__ __forceinline__ void finish_column(const AttnParams& p, float4 o, float lsum, bool on, bool has_keys, uint32_t col, uint32_t d4,
                                              const uint32_t* col_row, const uint32_t* col_orow, const uint32_t* col_head, bool report) {
  const bool good = lsum > 0.0f && isfinite(lsum);
  const float inv = good ? __frcp_rn(lsum) : 0.0f;
  float4 r = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  if (!good) r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (!good && on && has_keys && report) atomicCAS(p.fault, FAULT_NONE, FAULT_NONFINITE);
  if (on) *reinterpret_cast<float4*>(p.out + (uint64_t)col_row[col] * D + 4 * d4) = r;
  if (p.image) {
    const uint32_t irow = on ? col_orow[col] : 0, kb = on ? (col_head[col] * (D / 4) + d4) >> 3 : 0;
    if (p.image_dtype == AION_CUDA_DTYPE_Q8_0) quantize_store_block_8lanes<AION_CUDA_DTYPE_Q8_0>(r, d4 & 7, on, p.image, p.image_layout, irow, kb);
    else quantize_store_block_8lanes<AION_CUDA_DTYPE_Q4_0>(r, d4 & 7, on, p.image, p.image_layout, irow, kb);
  }
}

}  // namespace aion
