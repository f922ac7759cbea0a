// Quantized KV caches: rows are quantized as they are appended, logical steps are read back as values, and the
// projection's heads are normed, rotated and appended in one pass.
//
// A cache row of a head is D / 32 blocks of the weight formats: q8_0 (f16 scale, 32 int8) or q4_0 (f16 scale,
// 16 bytes of nibbles). The codes are those of aion_cuda_quantize, so this file is compiled without FMA
// contraction too. All three steps move each byte once and compute little: HBM bounds the large ones, the
// launch and one trip to memory the small ones.
#include <cmath>

#include "cache_geom.cuh"
#include "common.cuh"
#include "ptx.cuh"
#include "quant_device.cuh"

namespace aion {

namespace {

constexpr uint32_t FULL = 0xFFFFFFFFu;

// ---- the block quantizer, eight lanes to a block ------------------------------------------------
// Lane i of eight (i = lane & 7) holds values 4i .. 4i + 3 of a block. Returns the block's f16 scale and this
// lane's codes: q8_0 four bytes, q4_0 four nibbles. Operation for operation the block quantizer of quant.cu.
// All lanes of a warp call it together.
template <int DT>
__device__ __forceinline__ uint32_t quantize_4(const float (&v)[4], uint16_t* scale_bits) {
  float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
  amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 2));
  amax = fmaxf(amax, __shfl_xor_sync(FULL, amax, 4));
  uint32_t codes = 0;
  if (DT == AION_CUDA_DTYPE_Q8_0) {
    const float scale = amax == 0.0f ? 1.0f : __fdiv_rn(amax, 127.0f);
    const __half sh = __float2half_rn(scale);
    *scale_bits = __half_as_ushort(sh);
    const float eff = __half2float(sh);
    const float inv = (amax == 0.0f || eff == 0.0f) ? 0.0f : __fdiv_rn(1.0f, eff);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int q = max(-128, min(127, (int)roundf(__fmul_rn(v[j], inv))));
      codes |= ((uint32_t)q & 0xFFu) << (8 * j);
    }
  } else {
    const float scale = amax == 0.0f ? 1.0f : __fdiv_rn(amax, 7.0f);
    *scale_bits = __half_as_ushort(__float2half_rn(scale));
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int q = max(-8, min(7, (int)roundf(__fdiv_rn(v[j], scale)))) + 8;
      codes |= (uint32_t)q << (4 * j);
    }
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

// ---- append: eight lanes per block, blocks of all new rows in order -----------------------------
template <int DT, typename T>
__global__ void __launch_bounds__(256) append_quantized_kernel(uint8_t* __restrict__ cache, const T* __restrict__ rows,
                                                               const int32_t* __restrict__ end_index, CacheGeom g, uint32_t new_len,
                                                               uint32_t blocks_per_row, uint64_t nblocks, int* fault) {
  constexpr int BB = DT == AION_CUDA_DTYPE_Q8_0 ? Q8_BYTES : Q4_BYTES;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const uint32_t i = threadIdx.x & 7;
  const uint64_t step = (uint64_t)gridDim.x * (blockDim.x / 8);
  const uint64_t first = blockIdx.x * (uint64_t)(blockDim.x / 8) + threadIdx.x / 8;
  for (uint64_t base = first & ~3ull; base < nblocks; base += step) {   // the four groups of a warp leave together
    const uint64_t blk = base + (first & 3);
    const bool on = blk < nblocks;
    const uint64_t r = on ? blk / blocks_per_row : 0;
    const uint32_t in_row = on ? (uint32_t)(blk - r * blocks_per_row) : 0;
    const uint32_t b = (uint32_t)(r / new_len), t = (uint32_t)(r - (uint64_t)b * new_len);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (on)
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = (float)rows[blk * QK + 4 * i + j];
    bool bad = false;
    const int64_t row = on ? append_row(g, b, end_index[b], t, new_len, &bad) : -1;
    if (bad && i == 0) atomicCAS(fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
    uint16_t scale;
    const uint32_t codes = quantize_4<DT>(v, &scale);
    if (row >= 0) store_block_part<DT>(cache + ((uint64_t)row * blocks_per_row + in_row) * BB, i, codes, scale);
  }
}

// ---- read: values of logical steps -----------------------------------------------------------------
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

// One thread per value.
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
    const ReadSpan s = read_span(g, start, lengths, b);
    const uint64_t step = (uint64_t)(start && !s.bad ? start[b] : 0) + t;
    bool bad = s.bad;
    float v = 0.0f;
    if (step >= s.lo && step < s.hi) {
      const int64_t row = cache_row(g, b, (uint32_t)step);
      if (row < 0) bad = true;
      else v = row_value<DT>(cache + (uint64_t)row * row_bytes, e);
    }
    if (bad) atomicCAS(fault, FAULT_NONE, FAULT_INVALID_ARGUMENT);
    out[i] = as_out<O>(v);
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

unsigned blocks_for(const AionCudaDevice* dev, uint64_t items, unsigned per_block) {
  const uint64_t want = ceil_div(items, (uint64_t)per_block), cap = (uint64_t)dev->sm_count * 16;
  return (unsigned)(want < cap ? want : cap);
}

template <typename T>
int32_t launch_append(AionCudaDevice* dev, const AionCudaSequenceAppend* s, uint8_t* cache, const T* rows, const int32_t* idx, const CacheGeom& g) {
  const uint64_t bpr = s->heads * s->head_dim / QK, nblocks = s->batch * s->new_len * bpr;
  const dim3 grid(blocks_for(dev, nblocks, 256 / 8)), block(256);
  if (s->dtype == AION_CUDA_DTYPE_Q8_0)
    AION_CUDA_TRY(launch_pdl(append_quantized_kernel<AION_CUDA_DTYPE_Q8_0, T>, grid, block, 0, dev->stream, cache, rows, idx, g, (uint32_t)s->new_len,
                             (uint32_t)bpr, nblocks, dev->fault_dev));
  else
    AION_CUDA_TRY(launch_pdl(append_quantized_kernel<AION_CUDA_DTYPE_Q4_0, T>, grid, block, 0, dev->stream, cache, rows, idx, g, (uint32_t)s->new_len,
                             (uint32_t)bpr, nblocks, dev->fault_dev));
  return AION_CUDA_OK;
}

template <typename O>
int32_t launch_read(AionCudaDevice* dev, const AionCudaSequenceRead* s, O* out, const uint8_t* cache, const int32_t* start, const int32_t* lengths,
                    const CacheGeom& g) {
  const uint64_t row_values = s->heads * s->head_dim, count = s->batch * s->out_len * row_values;
  const uint64_t row_bytes = cache_bytes(s->dtype, row_values);
  const dim3 grid(blocks_for(dev, count, 256)), block(256);
#define AION_READ(DT)                                                                                                          \
  AION_CUDA_TRY(launch_pdl(sequence_read_kernel<DT, O>, grid, block, 0, dev->stream, out, cache, start, lengths, g, (uint32_t)s->out_len, \
                           (uint32_t)row_values, row_bytes, count, dev->fault_dev))
  switch (s->dtype) {
    case AION_CUDA_DTYPE_F32: AION_READ(AION_CUDA_DTYPE_F32); break;
    case AION_CUDA_DTYPE_F16: AION_READ(AION_CUDA_DTYPE_F16); break;
    case AION_CUDA_DTYPE_Q8_0: AION_READ(AION_CUDA_DTYPE_Q8_0); break;
    default: AION_READ(AION_CUDA_DTYPE_Q4_0); break;
  }
#undef AION_READ
  return AION_CUDA_OK;
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
  if (int32_t st = dev->make_current()) return st;
  uint8_t *cache, *nk;
  const int32_t* idx;
  if (int32_t st = resolve(s->cache, cache_bytes(s->dtype, rows * row_values), "sequence_append.cache", &cache)) return st;
  const uint64_t eb = s->new_dtype == AION_CUDA_DTYPE_F32 ? 4 : 2;
  if (int32_t st = resolve(s->new_kv, s->batch * s->new_len * row_values * eb, "sequence_append.new_kv", &nk)) return st;
  if (int32_t st = resolve(s->end_index, s->batch * sizeof(int32_t), "sequence_append.end_index", &idx)) return st;
  if ((reinterpret_cast<uintptr_t>(cache) & 1) || (reinterpret_cast<uintptr_t>(nk) & (eb - 1)))
    return fail(AION_CUDA_INVALID_ARGUMENT, "%s: misaligned operand", what);
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
  if (int32_t st = dev->make_current()) return st;
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
  if (int32_t st = dev->make_current()) return st;
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
  p.len = (uint32_t)s->len, p.h_q = (uint32_t)s->h_q, p.h_kv = (uint32_t)s->h_kv, p.d = (uint32_t)d;
  p.ld = ld;
  p.rope_pairs = pf > (float)(d / 2) ? (uint32_t)(d / 2) : (uint32_t)pf;
  p.step = (float)std::pow((double)s->base_frequency, (double)(-2.0f / (float)d));
  p.scale_factor = s->scale_factor, p.eps = s->eps;
  p.k_dtype = s->k_dtype, p.v_dtype = s->v_dtype;
  p.fault = dev->fault_dev;
  const size_t smem = (d + NR_WARPS * d) * sizeof(float);
  AION_CUDA_TRY(launch_pdl(qk_norm_rope_append_kernel, dim3((unsigned)rows), dim3(NR_THREADS), smem, dev->stream, p));
  return AION_CUDA_OK;
}

}  // extern "C"
