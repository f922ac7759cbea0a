// `Attention` over a quantized KV cache: K and V are q8_0 / q4_0 blocks of 32 along the head dimension, kept
// contiguous, as a ring, or in pages.
//
// With k_t = c_t * s_t (integer codes times the block's f16 scale), for every query row
//   logit_t = scale * sum_blocks s_t[block] * (q[block] . c_t[block])      (optional soft cap)
//   out[block] = sum_t softmax_t * s_t[block] * c_t[block]
// over the keys [lo, hi) of the row's window; zeros for an empty range. The codes are exact in any float type
// and the scales in f32, so only the f32 sums round: the result is f32 attention over the dequantized cache.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <mutex>

#include "attention_qcache.cuh"

namespace aion {

namespace {

using namespace qcache;

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
  dev->debug_qcache = {AION_CUDA_QCACHE_KERNEL_ANY, 1u, 0u};
  return AION_CUDA_OK;
}

// ------------------------------------------------------------------------------------
// tensor-core kernel for few query columns (decode): head sizes 64, 128, 256
// ------------------------------------------------------------------------------------
// A CTA serves up to eight query columns of one kv head, a column being (query position, query head of the
// group), and a slice of the context; its four warps walk tiles of 16 keys on their own, each with a private
// ring of stages, so nothing in the loop waits for another warp. A tile's rows arrive as one TMA box of K and one
// of V (16 rows of the head's bytes, rounded out to 16-byte granules) where the rows of the cache begin on
// 16-byte boundaries, else by cp.async in pieces of D / 16 bytes.
//
//  * S^T[16 keys x 8] = C . Q^T on f16 m16n8k16: the codes are exact in f16, q is two f16 terms (22 bits, normed
//    by the column's largest value), and the products of one block of 32 dimensions are scaled by the block's
//    scale in f32. q4_0 codes are made the normal numbers n - 8: as the subnormals n * 2^-24 that a nibble IS in the low
//    bits of an f16 they would need no arithmetic, but a tensor core aligns its products by the exponent fields, where a
//    subnormal counts as 2^-14, and cuts the low bits of q off.
//  * The logits are transposed by movmatrix (two 16-bit halves each), so a lane holds one column's logits of the
//    keys that it needs as the B operand of the second product.
//  * O^T[D x 8] += V-codes^T . P'^T, P' = p * scale of (key, block) in f32, again two f16 terms, the
//    second one times 2^11 with a sum of its own. P' is scaled by a power of two that follows the largest V scale
//    met so far: it is below 2^15, and where keys or columns differ in size the second term still has eleven bits when the
//    first one is down to f16's subnormals (23 bits of a P' down to 2^-29 of the largest). The accumulators are moved over
//    when that power or a column's maximum grows.
//  * The context of a unit (one kv head's columns) is cut over clusters of up to eight CTAs. A cluster's sums meet
//    through distributed shared memory, every CTA adding up its share of the outputs; only units that several
//    clusters work on leave partial sums in global memory, for the last of them to arrive. (With one ticket per
//    CTA instead, that one CTA's trips to L2 cost 7 us of a 1024-key decode's 14.)
//  * With fewer units than the GPU holds CTAs, the clusters are dealt out in proportion to the keys that each
//    unit has: every CTA works out the same table from the lengths and finds its place in it.
//
// A lane reads a block pair's bytes where they lie: 2 x 18 (34) bytes are 9 (17) aligned words whose first and
// middle ones hold the scales, and the order of the dimensions inside a block is free as long as Q's order is
// the same. Rows are padded in shared memory to a pitch of 4 (mod 8) words, where no two lanes meet in a bank.
constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int COLS = 8;

template <int D, bool KQ8, bool VQ8>
struct DecodeGeom {
  using K = RowFmt<D, KQ8>;
  using V = RowFmt<D, VQ8>;
  static constexpr int STAGE = TK * (K::PITCH + V::PITCH);
  // CTAs an SM: two for D = 256 (registers), three below. STAGES_FIT: what their shares of shared memory hold.
  static constexpr int CTAS = D == 256 ? 2 : 3;
  static constexpr int STAGES_FIT = (D == 256 ? 95 : 63) * 1024 / (WARPS * STAGE);
  static constexpr int NST = STAGES_FIT > 8 ? 8 : STAGES_FIT;
  // Tiles that an iteration takes together (the softmax, the waits and the f32 additions are paid once for them):
  // two where the ring then still holds two more.
  static constexpr int TPI = NST >= 4 ? 2 : 1;
  static constexpr int AHEAD = NST - TPI;            // tiles under way while an iteration computes
  static constexpr int WS = COLS * D + 2 * COLS;     // floats of a warp's result: sums, maxima, weights
  static constexpr int RING = WARPS * NST * STAGE;
  static_assert(NST >= 2 && WARPS * WS * 4 <= RING, "ring");
  static constexpr int OFF_VS = RING;                                        // f32 [warp][block][keys of an iteration]: V scales
  static constexpr int OFF_Q = OFF_VS + WARPS * (D / QK) * TK * TPI * 4;     // uint4 [D / 16][32]: Q fragments; first f32 [8][D]: q
  static constexpr int OFF_META = OFF_Q + COLS * D * 4;                      // per column: row, first key, key end, output row, head, factor
  static constexpr int OFF_VALID = OFF_META + COLS * 24;                     // per warp and stage: which keys are there, the first of them
  static constexpr int OFF_BARS = OFF_VALID + WARPS * NST * 8;               // per warp and stage: the copies' barrier
  static constexpr int OFF_FLAGS = OFF_BARS + WARPS * NST * 8;
  static constexpr int SMEM = OFF_FLAGS + 32;
  static_assert(CTAS * (SMEM + 1024) <= 227 * 1024, "shared memory of an SM");
  static constexpr int OFF_RES = WARPS * WS * 4;     // f32 [8][D], maxima, weights: the CTA's result, in the drained ring
  static_assert(OFF_RES % 16 == 0 && OFF_RES + WS * 4 <= RING, "room for the result");
  static constexpr int MAX_ROW_UNITS = COLS * D;     // tile counts that fit where q will lie
};

// How the units are dealt to the clusters.
struct DecodeGrid {
  uint32_t cluster;      // CTAs of a cluster
  uint32_t clusters;     // launched
  uint32_t row_units;    // (request, block of positions) pairs
  uint32_t per_row;      // units of each: kv heads x head groups
  uint32_t least;        // tiles that a cluster takes at least, where there are as many
  uint32_t dealt;        // 1: in proportion to the keys; 0: cluster c is unit c
};

__device__ __forceinline__ uint32_t count_tiles(const AttnParams& p, const TileSpace& ts, uint32_t b, uint32_t l0) {
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  for (uint32_t l = l0; l < min(p.L, l0 + p.pos_per_tile); l++) {
    const KeyRange r = key_range(p, b, l);
    if (r.hi > r.lo) lo = min(lo, r.lo), hi = max(hi, r.hi);
  }
  const TileRange t = tiles_of_keys(ts, lo, hi);
  return t.end - t.first;
}

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool there) {
  const int n = there ? BYTES : 0;   // nothing is read and zeros are written where the key is not there
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
template <int D, bool KQ8, bool VQ8, bool TMA>
__global__ void __launch_bounds__(THREADS, DecodeGeom<D, KQ8, VQ8>::CTAS) attn_qcache_decode_kernel(
    const AttnParams p, const DecodeGrid dg, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v) {
  using G = DecodeGeom<D, KQ8, VQ8>;
  using KF = RowFmt<D, KQ8>;
  using VF = RowFmt<D, VQ8>;
  constexpr int NB = D / QK;          // blocks of a head row
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = ptx::smem_u32(smem);
  auto lds32 = [&](uint32_t at) { return *reinterpret_cast<const uint32_t*>(smem + at); };
  auto lds16 = [&](uint32_t at) { return (uint32_t)*reinterpret_cast<const uint16_t*>(smem + at); };
  auto lds_f2 = [&](uint32_t at) { return *reinterpret_cast<const float2*>(smem + at); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;

  uint32_t* col_row = reinterpret_cast<uint32_t*>(smem + G::OFF_META);  // (b*L + l)*Hq + head, NO_ROW: padding
  uint32_t* col_lo = col_row + COLS;
  uint32_t* col_hi = col_lo + COLS;
  uint32_t* col_orow = col_hi + COLS;
  uint32_t* col_head = col_orow + COLS;
  float* col_factor = reinterpret_cast<float*>(col_head + COLS);
  float* qs = reinterpret_cast<float*>(smem + G::OFF_Q);
  int* flags = reinterpret_cast<int*>(smem + G::OFF_FLAGS);   // [0] bad inputs, [1] last cluster of the unit

  const uint32_t bars = sbase + G::OFF_BARS + warp * (G::NST * 8);
  if (tid == 0) flags[0] = 0;
  if (TMA && lane == 0) {
    for (int s = 0; s < G::NST; s++) ptx::mbar_init(bars + 8 * s, 1);
    ptx::fence_barrier_init();
  }
  __syncthreads();
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  const TileSpace ts = tile_space(geom_of(p));
  // ---- this cluster's unit, and its place among the unit's clusters
  const uint32_t cluster = blockIdx.x / dg.cluster, rank = blockIdx.x - cluster * dg.cluster;
  uint32_t row_unit = cluster / dg.per_row, in_row = cluster - row_unit * dg.per_row, split = 0, nsplit = 1;
  if (dg.dealt) {
    uint32_t* tiles_of = reinterpret_cast<uint32_t*>(smem + G::OFF_Q);
    for (uint32_t r = tid; r < dg.row_units; r += THREADS) {
      const uint32_t rb = r / p.l_blocks;
      tiles_of[r] = count_tiles(p, ts, rb, (r - rb * p.l_blocks) * p.pos_per_tile);
    }
    __syncthreads();
    uint32_t sum = 0;
    for (uint32_t r = lane; r < dg.row_units; r += 32) sum += tiles_of[r];
    sum = __reduce_add_sync(FULL, sum);
    // The smallest quota of tiles, to a few parts in a hundred, for which no more clusters are wanted than there are.
    // (sum ceil(t / quota) <= sum t / quota + units, so the first upper end is one.)
    const uint32_t units = dg.row_units * dg.per_row, spare = dg.clusters - units;
    auto wanted = [&](uint32_t quota) {
      uint32_t n = 0;
      for (uint32_t r = lane; r < dg.row_units; r += 32) n += max(1u, (tiles_of[r] + quota - 1) / quota);
      return __reduce_add_sync(FULL, n) * dg.per_row;
    };
    uint32_t quota = 0x7FFFFFFFu;
    if (spare) {
      const uint64_t all = (uint64_t)sum * dg.per_row;
      uint32_t low = (uint32_t)min((uint64_t)0x3FFFFFFFu, all / dg.clusters);
      quota = (uint32_t)min((uint64_t)0x3FFFFFFFu, (all + spare - 1) / spare) + 1;
      for (int i = 0; i < 4; i++) {
        const uint32_t mid = low + (quota - low) / 2;
        if (mid && wanted(mid) <= dg.clusters) quota = mid;
        else low = mid;
      }
      quota = max(dg.least, quota);
    }
    uint32_t before = 0;   // clusters of the row units before this batch of 32
    bool found = false;
    for (uint32_t r0 = 0; r0 < dg.row_units; r0 += 32) {
      const uint32_t r = r0 + lane;
      const uint32_t n = r < dg.row_units ? max(1u, (tiles_of[r] + quota - 1) / quota) : 0;
      uint32_t upto = n * dg.per_row;   // inclusive sum over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(FULL, upto, o);
        if (lane >= o) upto += x;
      }
      const uint32_t end = before + upto, mine = __ballot_sync(FULL, cluster < end);
      if (mine && !found) {   // the first lane whose clusters reach beyond this one's number
        const int owner = __ffs(mine) - 1;
        const uint32_t start = __shfl_sync(FULL, end - n * dg.per_row, owner);
        nsplit = __shfl_sync(FULL, n, owner);
        row_unit = r0 + owner;
        in_row = (cluster - start) / nsplit;
        split = (cluster - start) - in_row * nsplit;
        found = true;
        break;
      }
      before = __shfl_sync(FULL, end, 31);
    }
    if (!found) return;    // no unit wants this cluster: all of it leaves
    __syncthreads();       // the counts have been read, q may take their place
  }
  const uint32_t hkv = in_row / p.head_groups, hg = in_row - hkv * p.head_groups;
  const uint32_t b = row_unit / p.l_blocks;
  // (Later positions see more keys under a causal window: where units queue, the long ones begin first.)
  const uint32_t lb = dg.dealt ? row_unit - b * p.l_blocks : p.l_blocks - 1 - (row_unit - b * p.l_blocks);
  const uint32_t unit = row_unit * dg.per_row + in_row;
  const uint32_t group = p.Hq / p.Hkv;
  const uint32_t h0 = hkv * group + hg * 8;
  const uint32_t nh = min(8u, group - hg * 8);
  const uint32_t l0 = lb * p.pos_per_tile;
  // This warp's two columns of q are on their way while the ranges are worked out.
  float qv[COLS / WARPS][D / 32];
#pragma unroll
  for (int j = 0; j < COLS / WARPS; j++) {
    const uint32_t c = warp + j * WARPS, pl = c / p.col_heads, hh = c - pl * p.col_heads, l = l0 + pl;
    const bool on = pl < p.pos_per_tile && hh < nh && l < p.L;
    const uint64_t at = ((uint64_t)(b * p.L + l) * p.Hq + h0 + hh) * D + lane;
#pragma unroll
    for (int i = 0; i < D / 32; i++) {
      qv[j][i] = 0.0f;
      if (on) qv[j][i] = p.q_dtype == AION_CUDA_DTYPE_F32 ? static_cast<const float*>(p.q)[at + 32 * i] : __half2float(static_cast<const __half*>(p.q)[at + 32 * i]);
    }
  }
  if (tid < COLS) {
    const uint32_t pl = tid / p.col_heads, hh = tid - pl * p.col_heads, l = l0 + pl;
    uint32_t row = NO_ROW, lo = 0, hi = 0;
    if (pl < p.pos_per_tile && hh < nh && l < p.L) {
      const KeyRange kr = key_range(p, b, l);
      if (kr.bad) flags[0] = 1;
      row = (b * p.L + l) * p.Hq + h0 + hh;
      lo = kr.lo, hi = kr.hi;
    }
    col_row[tid] = row, col_lo[tid] = lo, col_hi[tid] = hi;
    col_orow[tid] = b * p.L + l, col_head[tid] = h0 + hh;
  }
  __syncthreads();
  if (flags[0] && tid == 0) atomicExch(p.fault, FAULT_INVALID_ARGUMENT);
  // The union of the columns' ranges, and what all of them see.
  uint32_t u_lo = 0xFFFFFFFFu, u_hi = 0, all_lo = 0, all_hi = 0xFFFFFFFFu;
#pragma unroll
  for (int c = 0; c < COLS; c++) {
    const uint32_t lo = col_lo[c], hi = col_hi[c];
    if (hi > lo) u_lo = min(u_lo, lo), u_hi = max(u_hi, hi);
    if (col_row[c] != NO_ROW) all_lo = max(all_lo, lo), all_hi = min(all_hi, hi);
  }
  u_lo = min(u_lo, u_hi);
  const TileRange whole = tiles_of_keys(ts, u_lo, u_hi);
  const uint32_t parts = nsplit * dg.cluster, per = (whole.end - whole.first + parts - 1) / parts;
  const uint32_t my_first = (uint32_t)min((uint64_t)whole.end, whole.first + (uint64_t)(split * dg.cluster + rank) * per);
  const uint32_t tiles = min(whole.end - my_first, per);

  // ---- the warp's copies. Its n-th tile is one of TPI neighbours; the warps take such groups in turn.
  const uint64_t row0 = p.page_table ? 0 : (uint64_t)b * p.T;   // the request's first row, or the pool's
  const uint32_t ring = warp * (G::NST * G::STAGE);   // offsets into shared memory
  uint2* valid = reinterpret_cast<uint2*>(smem + G::OFF_VALID) + warp * G::NST;   // per stage: which keys are there, the first key
  // A box begins on a 16-byte boundary: the head's bytes are this far into each row.
  const uint32_t kshift = TMA ? (hkv * KF::BYTES) & 15 : 0, vshift = TMA ? (hkv * VF::BYTES) & 15 : 0;
  auto tile_of = [&](uint32_t n) { return ((n / G::TPI) * WARPS + warp) * G::TPI + n % G::TPI; };
  // Where a tile lies: its segment, counted on from the last tile's (a division costs as much as a block of keys),
  // and the raw entry of the page table, which is read a tile ahead of the copies and looked at only then.
  uint32_t seg = (my_first + tile_of(0)) / ts.per_seg, in_seg = my_first + tile_of(0) - seg * ts.per_seg, last_n = 0;
  int32_t next_page = 0;
  auto place = [&](uint32_t n) {
    in_seg += tile_of(n) - tile_of(last_n);
    last_n = n;
    while (in_seg >= ts.per_seg) in_seg -= ts.per_seg, seg++;
    if (p.page_table && tile_of(n) < tiles) next_page = __ldg(p.page_table + (uint64_t)b * p.pages_per_request + seg);
  };
  auto issue = [&](uint32_t n) {
    const uint32_t stage = n % G::NST;
    uint32_t count = tile_of(n) < tiles ? tile_rows(ts, in_seg) : 0;   // keys of the tile
    uint64_t row = count ? row0 + in_seg * TK : 0;
    if (p.page_table) {
      if (count && (next_page < 0 || (uint32_t)next_page >= p.pool_pages)) {
        if (lane == 0) atomicExch(p.fault, FAULT_INVALID_ARGUMENT);   // a page outside the pool: its keys are left out
        count = 0;
      }
      row += (uint64_t)(count ? next_page : 0) * p.page_tokens;
    }
    if (lane == 0) valid[stage] = make_uint2((1u << count) - 1, seg * ts.seg_len + in_seg * TK);
    const uint32_t dst = sbase + ring + stage * G::STAGE, vdst = dst + TK * KF::PITCH;
    if constexpr (TMA) {
      if (lane == 0) {
        const uint32_t bar = bars + 8 * stage;
        ptx::mbar_arrive_expect_tx(bar, count ? (uint32_t)G::STAGE : 0u);
        if (count && !(p.drop_first && n == 0)) {
          ptx::tma_load_2d(dst, &tmap_k, (int)((hkv * KF::BYTES) / 16 * 2), (int)row, bar);
          ptx::tma_load_2d(vdst, &tmap_v, (int)((hkv * VF::BYTES) / 16 * 2), (int)row, bar);
        }
      }
    } else {
      const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + (row * p.Hkv + hkv) * KF::BYTES;
      const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + (row * p.Hkv + hkv) * VF::BYTES;
      // Where the key is not there the address is the first row's, and nothing is read from it.
#pragma unroll
      for (int i = 0; i < (TK * KF::CHUNKS + 31) / 32; i++) {
        const uint32_t idx = lane + 32 * i, key = idx / KF::CHUNKS, c = idx - key * KF::CHUNKS;
        if (idx < TK * KF::CHUNKS)
          cp_async<KF::CHUNK>(dst + key * KF::PITCH + c * KF::CHUNK, kbase + (key < count ? (uint64_t)key * (p.Hkv * KF::BYTES) + c * KF::CHUNK : 0), key < count);
      }
#pragma unroll
      for (int i = 0; i < (TK * VF::CHUNKS + 31) / 32; i++) {
        const uint32_t idx = lane + 32 * i, key = idx / VF::CHUNKS, c = idx - key * VF::CHUNKS;
        if (idx < TK * VF::CHUNKS)
          cp_async<VF::CHUNK>(vdst + key * VF::PITCH + c * VF::CHUNK, vbase + (key < count ? (uint64_t)key * (p.Hkv * VF::BYTES) + c * VF::CHUNK : 0), key < count);
      }
      cp_commit();
    }
  };
  const uint32_t groups = (tiles + G::TPI - 1) / G::TPI;
  const uint32_t iters = groups > (uint32_t)warp ? (groups - warp + WARPS - 1) / WARPS : 0;
  const uint32_t mine = iters * G::TPI;   // the last of them may lie behind the end: no key of it is there
  place(0);
#pragma unroll
  for (int n = 0; n < G::AHEAD; n++) {
    if ((uint32_t)n < mine) {
      issue(n);
      place(n + 1);
    } else if (!TMA) {
      cp_commit();
    }
  }

  // ---- q: normed by the column's largest value to [2^13, 2^14)
#pragma unroll
  for (int j = 0; j < COLS / WARPS; j++) {
    const int c = warp + j * WARPS;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 32; i++) top = fmaxf(top, fabsf(qv[j][i]));
    uint32_t e = __reduce_max_sync(FULL, __float_as_uint(top)) >> 23;     // biased exponent
    if (e == 255) e = 127;                                                // not finite: the logits will not be either
    e = max(e, 40u);                                                      // far below any logit that matters
    const float up = __uint_as_float((127u + 13u + 127u - e) << 23);      // 2^(13 - (e - 127)), e >= 40
#pragma unroll
    for (int i = 0; i < D / 32; i++) qs[c * D + lane + 32 * i] = qv[j][i] * up;
    if (lane == 0) col_factor[c] = p.scale * __uint_as_float((e - 13u) << 23);
  }
  __syncthreads();
  // Q^T as the B operand: this lane's column g, the dimensions of word t.
  // Every warp makes a part of the fragments for all.
  uint4 made[NB / WARPS > 0 ? NB / WARPS : 1][2];
#pragma unroll
  for (int j = 0; j < (NB + WARPS - 1) / WARPS; j++) {
    const int blk = warp + j * WARPS;
    if (blk < NB) {
#pragma unroll
      for (int m = 0; m < 2; m++) {
        uint32_t hl[2][2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
          float x[2];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            int dim;
            if (KQ8) dim = pair_byte(true, blk & 1, t + 4 * m, 2 * r + h);
            else dim = 2 * pair_byte(false, blk & 1, t, m + 2 * h) + r;      // nibbles (2m + r, 2m + r + 4): bytes m, m + 2
            x[h] = qs[g * D + blk * QK + dim];
          }
          split2(x[0], x[1], &hl[0][r], &hl[1][r]);
        }
        made[j][m] = make_uint4(hl[0][0], hl[0][1], hl[1][0], hl[1][1]);
      }
    }
  }
  __syncthreads();   // q has been read: the fragments take its place
  uint4* qfrag = reinterpret_cast<uint4*>(smem + G::OFF_Q);
#pragma unroll
  for (int j = 0; j < (NB + WARPS - 1) / WARPS; j++) {
    const int blk = warp + j * WARPS;
    if (blk < NB) qfrag[(2 * blk) * 32 + lane] = made[j][0], qfrag[(2 * blk + 1) * 32 + lane] = made[j][1];
  }
  __syncthreads();
  // With a soft cap the logits are wanted first; else they go straight to base 2.
  const float to_base2 = p.soft_cap > 0.0f ? 1.0f : LOG2E, inv_cap = p.soft_cap > 0.0f ? inverse_cap(p.soft_cap) : 0.0f;
  const float f0 = col_factor[2 * t] * to_base2, f1 = col_factor[2 * t + 1] * to_base2;
  const uint32_t lo_g = col_lo[g], hi_g = col_hi[g];

  float acc[D / 16][4];
#pragma unroll
  for (int i = 0; i < D / 16; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[i][e] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;     // column g; l_run: this lane's keys only
  uint32_t e_run = 0;                        // exponent field of the largest V scale so far
  constexpr int TPI = G::TPI, KI = TK * TPI;     // keys of an iteration
  const uint32_t vs = G::OFF_VS + warp * (NB * KI * 4);
  const uint32_t first_sel = t ? 0x3210u : 0x5432u, first_sel_v = g ? 0x3210u : 0x5432u;

  for (uint32_t it = 0; it < iters; it++) {
    // ---- the tiles of this iteration; those AHEAD of it set out
#pragma unroll
    for (int j = 0; j < TPI; j++) {
      const uint32_t n = it * TPI + G::AHEAD + j;
      if (n < mine) {
        issue(n);
        place(n + 1);
      } else if (!TMA) {
        cp_commit();
      }
    }
    if constexpr (TMA) {
      __syncwarp();
      bool landed = true;
#pragma unroll
      for (int j = 0; j < TPI; j++) {
        const uint32_t n = it * TPI + j;
        landed = landed && ptx::mbar_wait_bounded(bars + 8 * (n % G::NST), (n / G::NST) & 1, p.wait_limit);
      }
      if (!__all_sync(FULL, landed)) {
        if (lane == 0) atomicExch(p.fault, FAULT_WAIT_EXPIRED);
        // what is still under way lands before the ring is used for the merge
        for (uint32_t n = it * TPI; n < min(mine, it * TPI + (uint32_t)G::NST); n++) ptx::mbar_wait_bounded(bars + 8 * (n % G::NST), (n / G::NST) & 1, p.wait_limit);
        break;
      }
    } else {
      cp_wait<G::AHEAD>();
      __syncwarp();
    }
    uint32_t at[TPI], key0[TPI], there = 0;   // offset of a tile's K rows, its first key; which keys are there
    // Some column does not see some row of the tiles: what lies there (rows past the end, of other requests,
    // whatever a page holds) must not reach it, not even as 0 x infinity.
    bool partial = false;
#pragma unroll
    for (int j = 0; j < TPI; j++) {
      const uint32_t stage = (it * TPI + j) % G::NST;
      const uint2 v = valid[stage];
      at[j] = ring + stage * G::STAGE;
      key0[j] = v.y;
      there |= v.x << (TK * j);
      partial |= v.x != 0xFFFFu || v.y < all_lo || v.y + TK > all_hi;
    }

    // ---- V scales as f32, times 2^(29 - E) of the largest exponent so far. One that is not finite becomes 0 here and
    // makes the sums that it belongs to NaN below.
    uint32_t sc[NB * KI / 32], top = 0;
    bool weird = false;
#pragma unroll
    for (int j = 0; j < NB * KI / 32; j++) {
      const uint32_t e = lane + 32 * j, blk = e / KI, k = e % KI;
      sc[j] = lds16(at[TPI == 2 ? (k >> 4) : 0] + TK * KF::PITCH + vshift + (k & 15) * VF::PITCH + blk * VF::BB);
      if (partial) {   // only keys that some column sees
        const uint32_t key = key0[TPI == 2 ? (k >> 4) : 0] + (k & 15);
        if (!((there >> k) & 1) || key < u_lo || key >= u_hi) sc[j] = 0;
      }
      if ((sc[j] & 0x7FFFu) >= 0x7C00u) sc[j] = 0, weird = true;
      top = max(top, sc[j] & 0x7FFFu);
    }
    const uint32_t e_new = max(e_run, __reduce_max_sync(FULL, top) >> 10);
    const float vmul = __uint_as_float((127u + 29u - e_new) << 23);
#pragma unroll
    for (int j = 0; j < NB * KI / 32; j++) *reinterpret_cast<float*>(smem + vs + (lane + 32 * j) * 4) = half_bits(sc[j]) * vmul;
    weird = __any_sync(FULL, weird);
    __syncwarp();

    // ---- S^T: 16 keys x 8 columns for each tile
    float s[TPI][4];
#pragma unroll
    for (int j = 0; j < TPI; j++) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
    for (int pr = 0; pr < NB / 2; pr++) {
      uint32_t qh[4][2], ql[4][2];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const uint4 f = qfrag[(4 * pr + i) * 32 + lane];
        qh[i][0] = f.x, qh[i][1] = f.y, ql[i][0] = f.z, ql[i][1] = f.w;
      }
#pragma unroll
      for (int j = 0; j < TPI; j++) {
        uint32_t a[2][2][4];                   // [block of the pair][MMA][operand]
        float sl[2], sh[2];                    // scales of keys g, g + 8
#pragma unroll
        for (int half = 0; half < 2; half++) {
          const uint32_t row = at[j] + kshift + (g + 8 * half) * KF::PITCH + pr * 2 * KF::BB;
          const uint32_t w0 = lds32(row), wm = lds32(row + (KQ8 ? 32 : 16)), wt = lds32(row + 4 * t);
          const uint32_t first = __byte_perm(wt, wm, first_sel);
          if (KQ8) {
            unpack_q8(first, &a[0][0][half], &a[0][0][2 + half]);
            unpack_q8(lds32(row + 16 + 4 * t), &a[0][1][half], &a[0][1][2 + half]);
            unpack_q8(lds32(row + 36 + 4 * t), &a[1][0][half], &a[1][0][2 + half]);
            unpack_q8(lds32(row + 52 + 4 * t), &a[1][1][half], &a[1][1][2 + half]);
          } else {
            uint32_t u[4];
            unpack_q4(first, u);
            a[0][0][half] = u[0], a[0][0][2 + half] = u[1], a[0][1][half] = u[2], a[0][1][2 + half] = u[3];
            unpack_q4(lds32(row + 20 + 4 * t), u);
            a[1][0][half] = u[0], a[1][0][2 + half] = u[1], a[1][1][half] = u[2], a[1][1][2 + half] = u[3];
          }
          (half ? sh : sl)[0] = half_bits(w0 & 0xFFFFu), (half ? sh : sl)[1] = half_bits(wm >> 16);
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const int q = 2 * k;
          float c[4];
          mma_f16_from(c, a[k][0][0], a[k][0][1], a[k][0][2], a[k][0][3], ql[q][0], ql[q][1], 0.0f, 0.0f, 0.0f, 0.0f);
          mma_f16_from(c, a[k][1][0], a[k][1][1], a[k][1][2], a[k][1][3], ql[q + 1][0], ql[q + 1][1], c[0], c[1], c[2], c[3]);
          mma_f16_from(c, a[k][0][0], a[k][0][1], a[k][0][2], a[k][0][3], qh[q][0], qh[q][1], c[0], c[1], c[2], c[3]);
          mma_f16_from(c, a[k][1][0], a[k][1][1], a[k][1][2], a[k][1][3], qh[q + 1][0], qh[q + 1][1], c[0], c[1], c[2], c[3]);
          s[j][0] = fmaf(sl[k], c[0], s[j][0]);
          s[j][1] = fmaf(sl[k], c[1], s[j][1]);
          s[j][2] = fmaf(sh[k], c[2], s[j][2]);
          s[j][3] = fmaf(sh[k], c[3], s[j][3]);
        }
      }
    }
    // ---- logits, and their transpose: column g, keys 2t, 2t + 1, 2t + 8, 2t + 9 of each tile
    float y[4 * TPI];
#pragma unroll
    for (int j = 0; j < TPI; j++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t u = __float_as_uint(s[j][2 * h] * f0), w = __float_as_uint(s[j][2 * h + 1] * f1);
        const uint32_t low = movm(__byte_perm(u, w, 0x5410)), high = movm(__byte_perm(u, w, 0x7632));
        y[4 * j + 2 * h] = __uint_as_float(__byte_perm(low, high, 0x5410));
        y[4 * j + 2 * h + 1] = __uint_as_float(__byte_perm(low, high, 0x7632));
      }
    if (p.soft_cap > 0.0f) {
      cap_logits(y, p.soft_cap, inv_cap);
#pragma unroll
      for (int k = 0; k < 4 * TPI; k++) y[k] *= LOG2E;
    }
    if (partial) {
#pragma unroll
      for (int k = 0; k < 4 * TPI; k++) {
        const uint32_t kk = 2 * t + (k & 1) + 8 * (k >> 1), key = key0[k >> 2] + (kk & 15);
        if (!((there >> kk) & 1) || key < lo_g || key >= hi_g) y[k] = -INFINITY;
      }
    }
    float m_new = m_run;
#pragma unroll
    for (int k = 0; k < 4 * TPI; k++) m_new = fmaxf(m_new, y[k]);
    m_new = fmaxf(m_new, __shfl_xor_sync(FULL, m_new, 1));
    m_new = fmaxf(m_new, __shfl_xor_sync(FULL, m_new, 2));
    if (__any_sync(FULL, m_new > m_run || e_new > e_run)) {
      const float alpha = m_new > m_run ? ex2(m_run - m_new) : 1.0f;
      l_run *= alpha;
      const float down = __uint_as_float((127u + e_run - e_new) << 23);   // 2^(old - new)
      const float a0 = __shfl_sync(FULL, alpha, 8 * t) * down, a1 = __shfl_sync(FULL, alpha, 8 * t + 4) * down;
#pragma unroll
      for (int i = 0; i < D / 16; i++) acc[i][0] *= a0, acc[i][1] *= a1, acc[i][2] *= a0, acc[i][3] *= a1;
      m_run = m_new;
      e_run = e_new;
    }
    const float m_safe = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
    for (int k = 0; k < 4 * TPI; k++) {
      y[k] = ex2(y[k] - m_safe);
      l_run += y[k];
    }

    // ---- O^T += V^T . P'^T, block by block
#pragma unroll
      for (int blk = 0; blk < NB; blk++) {
        uint32_t bh[TPI][2], blw[TPI][2];
        uint32_t a[TPI][2][4];   // [tile][row tile][operand]: rows g and g + 8, key pairs (2t, 2t + 1) and (2t + 8, 2t + 9)
#pragma unroll
        for (int j = 0; j < TPI; j++) {
#pragma unroll
          for (int kp = 0; kp < 2; kp++) {
            const float2 v = lds_f2(vs + (blk * KI + j * TK + 2 * t + 8 * kp) * 4);
            const float2 w = mul2(make_float2(y[4 * j + 2 * kp], y[4 * j + 2 * kp + 1]), v);
            split2_scaled(w.x, w.y, &bh[j][kp], &blw[j][kp]);
            const uint32_t row = at[j] + TK * KF::PITCH + vshift + (2 * t + 8 * kp) * VF::PITCH;
            if (VQ8) {
              uint32_t x[2];
#pragma unroll
              for (int h = 0; h < 2; h++) {
                const uint32_t pos = row + h * VF::PITCH + (blk >> 1) * 2 * VF::BB;
                if (blk & 1) x[h] = lds32(pos + 36 + 4 * g);
                else x[h] = __byte_perm(lds32(pos + 4 * g), lds32(pos + 32), first_sel_v);
                x[h] ^= 0x80808080u;
              }
              const uint32_t lo2 = __byte_perm(x[0], x[1], 0x5140), hi2 = __byte_perm(x[0], x[1], 0x7362);
              a[j][0][2 * kp] = h2_add(__byte_perm(lo2, 0x64646464u, 0x4140), 0xE480E480u);
              a[j][0][2 * kp + 1] = h2_add(__byte_perm(lo2, 0x64646464u, 0x4342), 0xE480E480u);
              a[j][1][2 * kp] = h2_add(__byte_perm(hi2, 0x64646464u, 0x4140), 0xE480E480u);
              a[j][1][2 * kp + 1] = h2_add(__byte_perm(hi2, 0x64646464u, 0x4342), 0xE480E480u);
            } else {
              const uint32_t pos = row + blk * VF::BB + 2 + 2 * g;
              uint32_t u[4];
              unpack_q4(__byte_perm(lds16(pos), lds16(pos + VF::PITCH), 0x5410), u);
              a[j][0][2 * kp] = u[0], a[j][0][2 * kp + 1] = u[1], a[j][1][2 * kp] = u[2], a[j][1][2 * kp + 1] = u[3];
            }
          }
        }
        // The tensor core cuts its sums off instead of rounding them, always to the same side: over thousands of
        // keys that adds up. So an iteration is summed from zero and added in f32.
#pragma unroll
        for (int m = 0; m < 2; m++) {
          float o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ol[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int j = 0; j < TPI; j++) mma_f16_from(ol, a[j][m][0], a[j][m][1], a[j][m][2], a[j][m][3], blw[j][0], blw[j][1], ol[0], ol[1], ol[2], ol[3]);
#pragma unroll
          for (int j = 0; j < TPI; j++) mma_f16_from(o, a[j][m][0], a[j][m][1], a[j][m][2], a[j][m][3], bh[j][0], bh[j][1], o[0], o[1], o[2], o[3]);
          constexpr float down = 1.0f / LO_SCALE;
          const float2 x = fma2(make_float2(ol[0], ol[1]), make_float2(down, down), make_float2(o[0], o[1]));
          const float2 z = fma2(make_float2(ol[2], ol[3]), make_float2(down, down), make_float2(o[2], o[3]));
          add2(acc[2 * blk + m][0], acc[2 * blk + m][1], x.x, x.y);
          add2(acc[2 * blk + m][2], acc[2 * blk + m][3], z.x, z.y);
        }
      }
    if (weird) {
#pragma unroll
      for (int blk = 0; blk < NB; blk++) {
        bool met = false;   // column g gives weight to a key whose scale of this block is not finite
#pragma unroll
        for (int k = 0; k < 4 * TPI; k++) {
          const uint32_t kk = 2 * t + (k & 1) + 8 * ((k >> 1) & 1);
          const uint32_t bits = lds16(at[k >> 2] + TK * KF::PITCH + vshift + kk * VF::PITCH + blk * VF::BB) & 0x7FFFu;
          met |= bits >= 0x7C00u && y[k] > 0.0f;
        }
        const uint32_t who = __ballot_sync(FULL, met);
        const float n0 = (who >> (8 * t)) & 15 ? NAN : 0.0f, n1 = (who >> (8 * t + 4)) & 15 ? NAN : 0.0f;
#pragma unroll
        for (int m = 0; m < 2; m++) acc[2 * blk + m][0] += n0, acc[2 * blk + m][1] += n1, acc[2 * blk + m][2] += n0, acc[2 * blk + m][3] += n1;
      }
    }
    __syncwarp();   // the stages and the scales are free again
  }
  if (!TMA) cp_wait<0>();

  // ---- the four warps' sums meet
  l_run += __shfl_xor_sync(FULL, l_run, 1);
  l_run += __shfl_xor_sync(FULL, l_run, 2);
  __syncthreads();
  float* all = reinterpret_cast<float*>(smem);
  {
    float* mb = all + warp * G::WS;
    // 2^(E - 29): exact, but where the sum itself is below f32's normal range
    const float back = __uint_as_float((127u + e_run - 29u) << 23);
#pragma unroll
    for (int blk = 0; blk < NB; blk++)
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const int dim = blk * QK + (VQ8 ? pair_byte(true, blk & 1, g, 2 * m + r) : 4 * g + 2 * m + r);
          mb[(2 * t) * D + dim] = acc[2 * blk + m][2 * r] * back;
          mb[(2 * t + 1) * D + dim] = acc[2 * blk + m][2 * r + 1] * back;
        }
    if (t == 0) mb[COLS * D + g] = m_run, mb[COLS * D + COLS + g] = l_run;
  }
  __syncthreads();
  constexpr int C4 = COLS * D / 4 / THREADS;
  float* res = reinterpret_cast<float*>(smem + G::OFF_RES);   // [8][D], then maxima and weights
  const bool direct = nsplit * dg.cluster == 1;
#pragma unroll 1
  for (int c = 0; c < C4; c++) {
    const uint32_t idx4 = tid + c * THREADS, col = idx4 / (D / 4), d4 = idx4 % (D / 4);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; w++) M = fmaxf(M, all[w * G::WS + COLS * D + col]);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float lsum = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float mw = all[w * G::WS + COLS * D + col];
      const float f = mw == -INFINITY ? 0.0f : ex2(mw - M);
      const float4 x = *reinterpret_cast<const float4*>(all + w * G::WS + 4 * idx4);
      o.x += x.x * f, o.y += x.y * f, o.z += x.z * f, o.w += x.w * f;
      lsum += all[w * G::WS + COLS * D + COLS + col] * f;
    }
    if (direct) {
      finish_column<D>(p, o, lsum, col_row[col] != NO_ROW, col_hi[col] > col_lo[col], col, d4, col_row, col_orow, col_head, !flags[0]);
    } else {
      *reinterpret_cast<float4*>(res + 4 * idx4) = o;
      if (d4 == 0) res[COLS * D + col] = M, res[COLS * D + COLS + col] = lsum;
    }
  }
  if (direct) return;
  // ---- the cluster's: every CTA adds up its share of the outputs over all of them
  cluster_sync();
  constexpr int PP = D + 4;                   // a partial row: D sums, maximum, weight, pad
  const uint32_t share = COLS * D / 4 / dg.cluster;
  const uint32_t res_addr = sbase + G::OFF_RES;
  float* part = p.partial + (uint64_t)cluster * COLS * PP;
#pragma unroll 1
  for (uint32_t i = tid; i < (share + 31) / 32 * 32; i += THREADS) {   // whole warps: the image is made by eight lanes together
    const bool on4 = i < share;
    const uint32_t idx4 = rank * share + (on4 ? i : 0), col = idx4 / (D / 4), d4 = idx4 % (D / 4);
    const bool on = on4 && col_row[col] != NO_ROW;
    float m[8], l[8], M = -INFINITY, lsum = 0.0f;
    float4 v[8], o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < 8; k++) {
      m[k] = -INFINITY, l[k] = 0.0f, v[k] = o;
      if (k < (int)dg.cluster) {
        const uint32_t a = cluster_addr(res_addr, k);
        m[k] = ld_cluster_f(a + (COLS * D + col) * 4);
        l[k] = ld_cluster_f(a + (COLS * D + COLS + col) * 4);
        v[k] = ld_cluster_f4(a + 16 * idx4);
      }
      M = fmaxf(M, m[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float f = m[k] == -INFINITY ? 0.0f : ex2(m[k] - M);
      o.x += v[k].x * f, o.y += v[k].y * f, o.z += v[k].z * f, o.w += v[k].w * f;
      lsum += l[k] * f;
    }
    if (nsplit == 1) {
      finish_column<D>(p, o, lsum, on, col_hi[col] > col_lo[col], col, d4, col_row, col_orow, col_head, !flags[0]);
    } else if (on) {
      *reinterpret_cast<float4*>(part + col * PP + 4 * d4) = o;
      if (d4 == 0) *reinterpret_cast<float2*>(part + col * PP + D) = make_float2(M, lsum);
    }
  }
  if (nsplit > 1) __threadfence();
  cluster_sync();   // no CTA leaves, or looks for the others' sums, before all have read and written
  if (nsplit == 1) return;
  // ---- and the clusters' in the last of them to arrive
  if (rank == 0 && tid == 0) {
    __threadfence();
    const int prev = atomicAdd(p.tickets + unit, 1), last = prev == (int)nsplit - 1;
    if (last) p.tickets[unit] = 0;   // ready for the next launch
    for (uint32_t k = 0; k < dg.cluster; k++) st_cluster_u32(cluster_addr(sbase + G::OFF_FLAGS + 4, k), last);
  }
  cluster_sync();
  if (!flags[1]) return;
  __threadfence();
  const float* pu = p.partial + (uint64_t)(cluster - split) * COLS * PP;
#pragma unroll 1
  for (uint32_t i = tid; i < (share + 31) / 32 * 32; i += THREADS) {
    const bool on4 = i < share;
    const uint32_t idx4 = rank * share + (on4 ? i : 0), col = idx4 / (D / 4), d4 = idx4 % (D / 4);
    const bool on = on4 && col_row[col] != NO_ROW;
    float M = -INFINITY, lsum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t s0 = 0; s0 < nsplit; s0 += 8) {   // the loads of eight partial sums are under way together
      float2 ml[8];
      float4 v[8];
      float top = M;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        ml[k] = make_float2(-INFINITY, 0.0f), v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (on && s0 + k < nsplit) {
          const float* src = pu + ((uint64_t)(s0 + k) * COLS + col) * PP;
          ml[k] = __ldcg(reinterpret_cast<const float2*>(src + D));
          v[k] = __ldcg(reinterpret_cast<const float4*>(src + 4 * d4));
        }
      }
#pragma unroll
      for (int k = 0; k < 8; k++) top = fmaxf(top, ml[k].x);
      const float keep = M == -INFINITY ? 0.0f : ex2(M - top);
      o.x *= keep, o.y *= keep, o.z *= keep, o.w *= keep, lsum *= keep;
      M = top;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float f = ml[k].x == -INFINITY ? 0.0f : ex2(ml[k].x - M);
        o.x += v[k].x * f, o.y += v[k].y * f, o.z += v[k].z * f, o.w += v[k].w * f;
        lsum += ml[k].y * f;
      }
    }
    finish_column<D>(p, o, lsum, on, col_hi[col] > col_lo[col], col, d4, col_row, col_orow, col_head, !flags[0]);
  }
}

template <int D, bool KQ8, bool VQ8, bool TMA>
int32_t launch_decode_as(AionCudaDevice* dev, AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, uint64_t max_keys) {
  using G = DecodeGeom<D, KQ8, VQ8>;
  auto kernel = attn_qcache_decode_kernel<D, KQ8, VQ8, TMA>;
  // Clusters of 1, 2, 4 and 8 CTAs that the device holds at once; worked out once per device and instantiation.
  uint32_t resident[4];
  {
    static std::mutex mu;
    static uint32_t held[64][4] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (dev->ordinal < 0 || dev->ordinal >= 64) return fail(AION_CUDA_UNSUPPORTED, "attention: device %d", dev->ordinal);
    if (!held[dev->ordinal][0]) {
      AION_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM));
      prefer_max_shared(reinterpret_cast<const void*>(kernel));
      for (int i = 3; i >= 0; i--) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(8);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = G::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1u << i, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        AION_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
        held[dev->ordinal][i] = n > 0 ? (uint32_t)n : 1u;
      }
    }
    for (int i = 0; i < 4; i++) resident[i] = held[dev->ordinal][i];
  }
  DecodeGrid dg{};
  dg.row_units = p.B * p.l_blocks;
  dg.per_row = p.Hkv * p.head_groups;
  const uint64_t units = (uint64_t)dg.row_units * dg.per_row;
  // A cluster's CTAs add up their sums cheaply (2.5 us), so a unit gets as large a cluster as leaves every unit one and
  // every warp a tile. Where a warp has 16 tiles and more (30 us) it pays to deal smaller clusters out by the keys that
  // each unit has, although the table (3 us) and partial sums in global memory (4 us) come on top: 6 requests of
  // 25 941 to 65 536 keys take 194 us with a cluster of eight each, 152 us dealt; 64 of 512 to 2048 keys 24 and 27 us.
  const uint64_t tiles = (max_keys + TK - 1) / TK, per_warp = tiles * units / ((uint64_t)resident[0] * WARPS);
  const bool deal = per_warp >= 16 && units > 1;
  const uint64_t each = deal ? (per_warp >= 32 ? 8 : 4) : 1;   // clusters a unit, so that the shares come out even
  int lg = 0;
  while (lg < 3 && each * units <= resident[lg + 1] && tiles >= ((uint64_t)WARPS << (lg + 1))) lg++;
  if (dev->attn_split_override) for (lg = 0; lg < 3 && (2u << lg) <= dev->attn_split_override; lg++) {}
  dg.cluster = 1u << lg;
  // A single unit with more keys than one cluster should walk (four tiles a warp) takes several as well.
  dg.least = dg.cluster * WARPS * 4;
  dg.dealt = (deal || units == 1) && units < resident[lg] && dg.row_units <= (uint32_t)G::MAX_ROW_UNITS && tiles > dg.least;
  dg.clusters = dg.dealt ? resident[lg] : (uint32_t)units;
  if (dg.dealt) {
    if (int32_t st = dev->reserve_scratch((size_t)dg.clusters * COLS * (D + 4) * sizeof(float))) return st;
    if (int32_t st = dev->reserve_tickets(units)) return st;
    p.partial = static_cast<float*>(dev->lane_scratch());
    p.tickets = dev->lane_tickets();
  }
  if ((uint64_t)dg.clusters * dg.cluster > 0x7FFFFFFFull) return fail(AION_CUDA_UNSUPPORTED, "attention: too many rows");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(dg.clusters * dg.cluster);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = G::SMEM;
  cfg.stream = dev->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = dg.cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  static const bool no_pdl_main = std::getenv("AION_CUDA_NO_PDL_MAIN") != nullptr;  // tuning only
  cfg.numAttrs = no_pdl_main ? 1 : 2;
  AION_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p, dg, tk, tv));
  dev->debug_qcache = {TMA ? AION_CUDA_QCACHE_KERNEL_COLUMNS_BOXES : AION_CUDA_QCACHE_KERNEL_COLUMNS, dg.cluster, dg.dealt};
  return AION_CUDA_OK;
}

template <int D, bool KQ8, bool VQ8>
int32_t launch_decode(AionCudaDevice* dev, AttnParams& p, uint64_t max_keys, bool rows_kernel) {
  using KF = RowFmt<D, KQ8>;
  using VF = RowFmt<D, VQ8>;
  const uint64_t rows = p.page_table ? (uint64_t)p.pool_pages * p.page_tokens : (uint64_t)p.B * p.T;
  const uint64_t kw = (uint64_t)p.Hkv * KF::BYTES, vw = (uint64_t)p.Hkv * VF::BYTES;
  // Boxes need rows that begin on 16-byte boundaries.
  const bool boxes = ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | kw | vw) & 15) == 0 && rows < (1ull << 31);
  CUtensorMap tk{}, tv{};
  if (!boxes) return launch_decode_as<D, KQ8, VQ8, false>(dev, p, tk, tv, max_keys);
  const CUtensorMap* m;
  const uint64_t kd[2] = {kw, rows}, vd[2] = {vw, rows};
  const uint32_t kbox[2] = {KF::PITCH, TK}, vbox[2] = {VF::PITCH, TK};
  if (int32_t st = tensor_map_bytes(dev, p.k, 2, kd, &kw, kbox, &m)) return st;
  tk = *m;
  if (int32_t st = tensor_map_bytes(dev, p.v, 2, vd, &vw, vbox, &m)) return st;
  tv = *m;
  if (rows_kernel) return attention_qcache_rows(dev, p, tk, tv, max_keys);
  return launch_decode_as<D, KQ8, VQ8, true>(dev, p, tk, tv, max_keys);
}

}  // namespace

int32_t attention_qcache_launch(AionCudaDevice* dev, AttnParams& p, uint32_t flags) {
  const bool kq8 = p.k_dtype == AION_CUDA_DTYPE_Q8_0, vq8 = p.v_dtype == AION_CUDA_DTYPE_Q8_0;
  // The tensor-core kernel copies rows in pieces of D / 16 bytes and stores its output in 16 bytes.
  const uintptr_t kv = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
  const bool tensor = p.Dk == p.Dv && (p.Dk == 64 || p.Dk == 128 || p.Dk == 256) && (kv & (p.Dk / 16 - 1)) == 0 &&
                      (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && !(flags & AION_CUDA_ATTENTION_GENERIC);
  if (tensor) {
    const uint32_t group = p.Hq / p.Hkv;
    p.head_groups = (group + 7) / 8;
    p.col_heads = group < 8 ? group : 8;
    p.pos_per_tile = 8 / p.col_heads;
    if (p.pos_per_tile > p.L) p.pos_per_tile = p.L;
    p.l_blocks = (p.L + p.pos_per_tile - 1) / p.pos_per_tile;
    const uint64_t units = (uint64_t)p.B * p.l_blocks * p.Hkv * p.head_groups;
    if (units > 0x7FFFFFFF) return fail(AION_CUDA_UNSUPPORTED, "attention: too many rows");
    // Upper bound of the keys of a unit.
    uint64_t max_keys = p.T;
    const uint64_t span = (uint64_t)(p.win_chunk ? p.win_chunk : 1) + p.win_left + p.win_right + p.pos_per_tile;
    if (p.win_left != AION_CUDA_WINDOW_UNBOUNDED && p.win_right != AION_CUDA_WINDOW_UNBOUNDED && span < max_keys) max_keys = span;
    // Few columns at a time or 128 rows: by what each would cost. A unit of eight columns passes a key in 16, 24 or 31 ns
    // (D = 64, 128, 256) with all resident CTAs at work, after 8 us; a unit of 128 rows in 25, 34 or 51 ns, after 8, 10 or
    // 15 us and 1.1 us for each CTA of a cluster. (8 heads over 4 kv heads of 256: 32 positions of one request over 2048 keys
    // 17 us by columns, 40 us by rows; of eight requests over 4096 keys 130 and 72 us, 256 positions 846 and 231 us. 16 over 4
    // of 64: 16 and 23, 112 and 40, 616 and 232 us.)
    const int size = p.Dk == 64 ? 0 : p.Dk == 128 ? 1 : 2;
    constexpr double column_ns[3] = {16.0, 24.0, 31.0}, row_ns[3] = {25.0, 34.0, 51.0}, row_start[3] = {8.0, 10.0, 15.0};
    const double sms = (double)dev->sm_count, keys = (double)max_keys;
    const double columns_us = 8.0 + 1e-3 * column_ns[size] * keys * std::max(1.0 / 8.0, (double)units / (sms * (p.Dk == 256 ? 2.0 : 3.0)));
    const uint64_t blocks = (uint64_t)p.B * p.Hkv * (((uint64_t)p.L * group + 127) / 128);
    double rows_us = 1e30;
    for (uint64_t cluster = 1; cluster <= 8; cluster *= 2)
      rows_us = std::min(rows_us, row_start[size] + (cluster > 1 ? 1.1 * (double)cluster : 0.0) + 1e-3 * row_ns[size] * keys / (double)cluster * std::ceil((double)(blocks * cluster) / (sms * (cluster > 2 ? 0.85 : 1.0))));
    const bool rows_kernel = !p.image && p.L > 1 && !(flags & AION_CUDA_ATTENTION_ROW_UNITS) && ((flags & AION_CUDA_ATTENTION_BLOCKS) || rows_us < columns_us);
#define AION_QCACHE(D)                                                                                     \
  if (kq8) return vq8 ? launch_decode<D, true, true>(dev, p, max_keys, rows_kernel) : launch_decode<D, true, false>(dev, p, max_keys, rows_kernel); \
  return vq8 ? launch_decode<D, false, true>(dev, p, max_keys, rows_kernel) : launch_decode<D, false, false>(dev, p, max_keys, rows_kernel);
    switch (p.Dk) {
      case 64: AION_QCACHE(64)
      case 128: AION_QCACHE(128)
      default: AION_QCACHE(256)
    }
#undef AION_QCACHE
  }
  if (p.image) return fail(AION_CUDA_UNSUPPORTED, "attention: the output image is written by the tensor-core kernels only (Dk = Dv in {64, 128, 256}, aligned operands)");
  if (p.Dv > 32 * MAX_DV_PER_LANE || (p.Dk + ROW_WARPS * (p.Dv + 2)) * sizeof(float) > 48 * 1024)
    return fail(AION_CUDA_UNSUPPORTED, "attention: head dimensions %u / %u exceed the any-shape kernel", p.Dk, p.Dv);
  p.splits = 1;
  if (kq8) return vq8 ? launch_rows<true, true>(dev, p) : launch_rows<true, false>(dev, p);
  return vq8 ? launch_rows<false, true>(dev, p) : launch_rows<false, false>(dev, p);
}

}  // namespace aion
