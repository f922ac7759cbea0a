// `Attention` over a quantized KV cache for many query rows (prompts, several new rows per request): a CTA holds up to 128
// rows of one kv head, a row being (query position, query head of the group), sixteen to a warp, and streams the keys once
// for all of them.
//
//  * S[16 x 64] = Q . C^T and O[16 x D] += P' . V-codes on f16 m16n8k16 with the codes as exact f16 integers (see
//    attention_qcache.cu): q and P' = p * (V scale) are two f16 terms each, so the tensor pipe does 8 * rows * keys * D
//    operations for the 4 that f32 attention counts, and half its rate is the ceiling. Dequantized operands for tcgen05
//    would need two terms of K and V as well (three products each), and 128 x 256 queries in two terms fill the shared
//    memory that their tiles would need.
//  * The logits' fragment is the second product's A operand as it stands; only the scale of (key, block) is multiplied in
//    per block of 32 dimensions, before the split into two terms.
//  * Four warps turn the raw blocks into fragments of f16 codes, in the order in which the MMAs' lanes take them, and the
//    scales into f32; eight warps consume them, sixteen rows each. (With every warp unpacking for itself a tensor
//    instruction came with eight others, and the 1024-row chunk that takes XXX us took 721.) Two buffers of 32 keys lie
//    between the two sides; raw tiles arrive as TMA boxes of 16 rows. The consumers hold 216 registers, the unpacking
//    warps 72.
//  * A context too long for the few CTAs of a short prompt is cut over a cluster, whose CTAs add up their sums through
//    distributed shared memory.
#include <cmath>
#include <cstdlib>
#include <mutex>

#include "attention_qcache.cuh"

namespace aion {

namespace {

using namespace qcache;

constexpr int RW = 8;                 // consumer warps
constexpr int PW = 4;                 // unpacking warps
constexpr int RTHREADS = (RW + PW) * 32;
constexpr int ROWS = RW * 16;
constexpr int SUBS = 2;               // tiles of a stage
constexpr int SK = SUBS * TK;         // keys of a stage
constexpr int CONSUMER_REGS = 216, UNPACK_REGS = 72;
static_assert(CONSUMER_REGS * RW * 32 + UNPACK_REGS * PW * 32 <= 168 * RTHREADS, "the registers that the block is launched with");

struct RowsGrid {
  uint32_t cluster;      // CTAs that share a unit's keys
  uint32_t row_blocks;   // blocks of ROWS rows per (request, kv head)
  uint32_t rows;         // L * query heads of the group
};

template <int D, bool KQ8, bool VQ8>
struct RowsGeom {
  using K = RowFmt<D, KQ8>;
  using V = RowFmt<D, VQ8>;
  static constexpr int NB = D / QK;
  static constexpr int TILE = TK * (K::PITCH + V::PITCH);
  static constexpr int STAGE = SUBS * TILE;
  static constexpr int RAWS = D == 256 ? 1 : 2;                  // raw stages
  static constexpr int KFRAG = NB * (SK / 8) * 512, VFRAG = NB * SUBS * 1024, FRAG = KFRAG + VFRAG;
  static constexpr int OFF_QF = 0;                               // uint4 [warp][D / 16][hi, lo][32]; at the end f32 [ROWS][D]
  static constexpr int QF_BYTES = RW * (D / 16) * 2 * 512;
  static constexpr int OFF_FRAG = OFF_QF + QF_BYTES;             // uint4 [2][K: block, 8 keys][32], [V: block, 16 keys, half][32]
  static constexpr int OFF_RAW = OFF_FRAG + 2 * FRAG;
  static constexpr int OFF_KS = OFF_RAW + RAWS * STAGE;          // f32 [2][block][32]: K scales
  static constexpr int OFF_VS = OFF_KS + 2 * NB * SK * 4;        // f32 [2][block][32]: V scales, times 2^(29 - E)
  static constexpr int OFF_CI = OFF_VS + 2 * NB * SK * 4;        // f32 [warp][block][16]: -8 sum q
  static constexpr int OFF_STATS = OFF_CI + RW * NB * 16 * 4;    // f32 [2][ROWS]: the rows' maxima and weights, for the cluster
  static constexpr int OFF_ODD = OFF_STATS + 2 * ROWS * 4;       // u32 [2][block]: keys whose V scale is not finite
  static constexpr int OFF_RVALID = OFF_ODD + 2 * NB * 4;        // uint2 [RAWS][SUBS]: which keys are there, the first of them
  static constexpr int OFF_VALID = OFF_RVALID + RAWS * SUBS * 8; // the same for the fragments [2][SUBS], then [2] {exponent, any odd}
  static constexpr int OFF_BARS = OFF_VALID + 2 * SUBS * 8 + 2 * 8;   // raw full [2], fragments full [2], empty [2]
  static constexpr int OFF_FLAGS = OFF_BARS + 6 * 8;             // bad inputs, gave up, largest V scale, -, first key, key end
  static constexpr int SMEM = OFF_FLAGS + 32;
  static_assert(QF_BYTES == ROWS * D * 4 && OFF_RAW % 128 == 0 && SMEM <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void unpackers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(PW * 32) : "memory"); }

template <int D, bool KQ8, bool VQ8>
__global__ void __launch_bounds__(RTHREADS, 1) attn_qcache_rows_kernel(const AttnParams p, const RowsGrid rg, const __grid_constant__ CUtensorMap tmap_k,
                                                                      const __grid_constant__ CUtensorMap tmap_v) {
  using G = RowsGeom<D, KQ8, VQ8>;
  using KF = RowFmt<D, KQ8>;
  using VF = RowFmt<D, VQ8>;
  constexpr int NB = G::NB;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = ptx::smem_u32(smem);
  auto lds32 = [&](uint32_t at) { return *reinterpret_cast<const uint32_t*>(smem + at); };
  auto lds16 = [&](uint32_t at) { return (uint32_t)*reinterpret_cast<const uint16_t*>(smem + at); };
  auto lds_f2 = [&](uint32_t at) { return *reinterpret_cast<const float2*>(smem + at); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t raw_full = sbase + G::OFF_BARS, frag_full = raw_full + 16, frag_empty = raw_full + 32;
  volatile uint32_t* flags = reinterpret_cast<uint32_t*>(smem + G::OFF_FLAGS);
  uint2* raw_valid = reinterpret_cast<uint2*>(smem + G::OFF_RVALID);
  uint2* valid = reinterpret_cast<uint2*>(smem + G::OFF_VALID);       // [2][SUBS]
  uint2* summary = valid + 2 * SUBS;                                  // [2]
  uint32_t* odd = reinterpret_cast<uint32_t*>(smem + G::OFF_ODD);     // [2][NB]
  const bool consumer = warp < RW;

  if (tid == 0) {
    for (int s = 0; s < 2; s++) {
      ptx::mbar_init(raw_full + 8 * s, 1);
      ptx::mbar_init(frag_full + 8 * s, PW);
      ptx::mbar_init(frag_empty + 8 * s, RW);
    }
    flags[0] = flags[1] = flags[2] = flags[3] = flags[5] = 0;
    flags[4] = 0xFFFFFFFFu;
    ptx::fence_barrier_init();
  }
  __syncthreads();
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();

  // unit = (b, block of rows, kv head), blocks last first (they see most keys under a causal window); rank: its slice of the keys
  const uint32_t unit = blockIdx.x / rg.cluster, rank = blockIdx.x - unit * rg.cluster;
  const uint32_t hkv = unit % p.Hkv, bl = unit / p.Hkv, b = bl / rg.row_blocks, rb = rg.row_blocks - 1 - (bl - b * rg.row_blocks);
  const uint32_t group = p.Hq / p.Hkv;
  // Row r of the block: position and head of it, its row of q and out seen as [B * L * Hq, D]; NO_ROW beyond the last.
  auto row_of = [&](uint32_t r, uint32_t* l) -> uint32_t {
    const uint32_t i = rb * ROWS + r;
    *l = i / group;
    return i < rg.rows ? (b * p.L + *l) * p.Hq + hkv * group + (i - *l * group) : NO_ROW;
  };
  uint32_t my_row[2], lo[2], hi[2];   // rows g and g + 8 of the warp
  bool bad = false;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    uint32_t l;
    my_row[h] = consumer ? row_of(warp * 16 + g + 8 * h, &l) : NO_ROW;
    lo[h] = hi[h] = 0;
    if (my_row[h] != NO_ROW) {
      const KeyRange kr = key_range(p, b, l);
      bad |= kr.bad;
      lo[h] = kr.lo, hi[h] = kr.hi;
    }
  }
  if (bad) flags[0] = 1;
  // What some row of the warp sees, and what all of its rows see.
  uint32_t w_lo = 0xFFFFFFFFu, w_hi = 0, w_all_lo = 0, w_all_hi = 0xFFFFFFFFu;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    if (hi[h] > lo[h]) w_lo = min(w_lo, lo[h]), w_hi = max(w_hi, hi[h]);
    if (my_row[h] != NO_ROW) w_all_lo = max(w_all_lo, lo[h]), w_all_hi = min(w_all_hi, hi[h]);
  }
  w_lo = __reduce_min_sync(FULL, w_lo), w_hi = __reduce_max_sync(FULL, w_hi);
  w_all_lo = __reduce_max_sync(FULL, w_all_lo), w_all_hi = __reduce_min_sync(FULL, w_all_hi);
  if (lane == 0 && w_hi > 0) atomicMin(const_cast<uint32_t*>(flags) + 4, w_lo), atomicMax(const_cast<uint32_t*>(flags) + 5, w_hi);
  __syncthreads();
  if (flags[0] && tid == 0) atomicExch(p.fault, FAULT_INVALID_ARGUMENT);
  const uint32_t u_hi = flags[5], u_lo = min(flags[4], u_hi);
  const TileSpace ts = tile_space(p);
  const TileRange whole = tiles_of_keys(ts, u_lo, u_hi);
  uint32_t per = (whole.end - whole.first + rg.cluster - 1) / rg.cluster;
  per = (per + SUBS - 1) / SUBS * SUBS;
  const uint32_t my_first = (uint32_t)min((uint64_t)whole.end, whole.first + (uint64_t)rank * per);
  const uint32_t tiles = min(whole.end - my_first, per), stages = (tiles + SUBS - 1) / SUBS;

  float acc[NB][4][4];   // [block][8 dimensions][row g: 2, row g + 8: 2]
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
  uint32_t e_run = 0;

  if (!consumer) {
    // ================ raw blocks to fragments ================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(UNPACK_REGS));
    const int ptid = tid - RW * 32, pwarp = warp - RW;
    const uint64_t row0 = p.page_table ? 0 : (uint64_t)b * p.T;
    const uint32_t kshift = (hkv * KF::BYTES) & 15, vshift = (hkv * VF::BYTES) & 15;
    // The first of these threads brings the raw stages; the page numbers of the next one are read a stage ahead.
    uint32_t seg = my_first / ts.per_seg, in_seg = my_first - seg * ts.per_seg;
    uint32_t next_seg[SUBS], next_in[SUBS];
    int32_t next_page[SUBS];
    auto place = [&](uint32_t stage) {
#pragma unroll
      for (int s = 0; s < SUBS; s++) {
        next_seg[s] = seg, next_in[s] = in_seg, next_page[s] = 0;
        if (p.page_table && stage * SUBS + s < tiles) next_page[s] = __ldg(p.page_table + (uint64_t)b * p.pages_per_request + seg);
        if (++in_seg >= ts.per_seg) in_seg = 0, seg++;
      }
    };
    auto issue = [&](uint32_t stage) {
      const uint32_t st = stage % G::RAWS, bar = raw_full + 8 * st, dst = sbase + G::OFF_RAW + st * G::STAGE;
      uint32_t count[SUBS], bytes = 0;
      uint64_t row[SUBS];
#pragma unroll
      for (int s = 0; s < SUBS; s++) {
        count[s] = stage * SUBS + s < tiles ? min((uint32_t)TK, ts.seg_len - next_in[s] * TK) : 0;
        row[s] = row0 + next_in[s] * TK;
        if (p.page_table) {
          if (count[s] && (next_page[s] < 0 || (uint32_t)next_page[s] >= p.pool_pages)) {
            atomicExch(p.fault, FAULT_INVALID_ARGUMENT);   // a page outside the pool: its keys are left out
            count[s] = 0;
          }
          row[s] += (uint64_t)(count[s] ? next_page[s] : 0) * p.page_tokens;
        }
        raw_valid[st * SUBS + s] = make_uint2((1u << count[s]) - 1, next_seg[s] * ts.seg_len + next_in[s] * TK);
        if (count[s]) bytes += G::TILE;
      }
      ptx::mbar_arrive_expect_tx(bar, bytes);
      if (p.drop_first && stage == 0) return;
#pragma unroll
      for (int s = 0; s < SUBS; s++)
        if (count[s]) {
          ptx::tma_load_2d(dst + s * G::TILE, &tmap_k, (int)((hkv * KF::BYTES) / 16 * 2), (int)row[s], bar);
          ptx::tma_load_2d(dst + s * G::TILE + TK * KF::PITCH, &tmap_v, (int)((hkv * VF::BYTES) / 16 * 2), (int)row[s], bar);
        }
    };
    if (ptid == 0)
      for (uint32_t s = 0; s < min(stages, (uint32_t)G::RAWS); s++) place(s), issue(s);
    if (ptid == 0) place(G::RAWS);
    const uint32_t first_sel = t ? 0x3210u : 0x5432u, first_sel_v = g ? 0x3210u : 0x5432u;
    for (uint32_t it = 0; it < stages; it++) {
      const uint32_t buf = it & 1, raw = G::OFF_RAW + (it % G::RAWS) * G::STAGE, frag = G::OFF_FRAG + buf * G::FRAG + lane * 16;
      bool ok = ptx::mbar_wait_bounded(raw_full + 8 * (it % G::RAWS), (it / G::RAWS) & 1, p.wait_limit);
      if (it >= 2) ok = ptx::mbar_wait_bounded(frag_empty + 8 * buf, (it / 2 - 1) & 1, p.wait_limit) && ok;
      if (!ok) flags[1] = 1;
      // ---- scales
      constexpr int PER = (NB * SK + PW * 32 - 1) / (PW * 32);
      uint32_t vsc[PER], top = 0;
#pragma unroll
      for (int j = 0; j < PER; j++) {
        const uint32_t blk = pwarp + PW * j;   // a warp takes the 32 keys of a block
        vsc[j] = 0;
        if (blk >= NB) break;
        const uint32_t at = raw + (lane / TK) * G::TILE;
        const float ks = half_bits(lds16(at + kshift + (lane % TK) * KF::PITCH + blk * KF::BB));
        *reinterpret_cast<float*>(smem + G::OFF_KS + ((buf * NB + blk) * SK + lane) * 4) = ks;
        vsc[j] = lds16(at + TK * KF::PITCH + vshift + (lane % TK) * VF::PITCH + blk * VF::BB);
        const uint2 v = raw_valid[(it % G::RAWS) * SUBS + lane / TK];
        const uint32_t key = v.y + lane % TK;
        if (!((v.x >> (lane % TK)) & 1) || key < u_lo || key >= u_hi) vsc[j] = 0;   // no row sees it
        const uint32_t not_finite = __ballot_sync(FULL, (vsc[j] & 0x7FFFu) >= 0x7C00u);
        if ((vsc[j] & 0x7FFFu) >= 0x7C00u) vsc[j] = 0;
        if (lane == 0) odd[buf * NB + blk] = not_finite;
        top = max(top, vsc[j] & 0x7FFFu);
      }
      top = __reduce_max_sync(FULL, top);
      if (lane == 0) atomicMax(const_cast<uint32_t*>(flags) + 2, top);
      unpackers_sync();
      if (flags[1]) {
        if (ptid == 0) atomicExch(p.fault, FAULT_WAIT_EXPIRED);
        for (uint32_t s = it; s < min(stages, it + G::RAWS); s++) ptx::mbar_wait_bounded(raw_full + 8 * (s % G::RAWS), (s / G::RAWS) & 1, p.wait_limit);
        break;
      }
      const uint32_t e_new = flags[2] >> 10;   // the largest exponent so far
      const float vmul = __uint_as_float((127u + 29u - e_new) << 23);
#pragma unroll
      for (int j = 0; j < PER; j++) {
        const uint32_t blk = pwarp + PW * j;
        if (blk < NB) *reinterpret_cast<float*>(smem + G::OFF_VS + ((buf * NB + blk) * SK + lane) * 4) = half_bits(vsc[j]) * vmul;
      }
      if (ptid == 0) {
        uint32_t any = 0;
        for (int i = 0; i < NB; i++) any |= odd[buf * NB + i];
        summary[buf] = make_uint2(e_new, any);
        for (int s = 0; s < SUBS; s++) valid[buf * SUBS + s] = raw_valid[(it % G::RAWS) * SUBS + s];
      }
      // ---- K: the B operand of 8 keys x 32 dimensions
      for (int n = pwarp; n < NB * (SK / 8); n += PW) {
        const uint32_t blk = n / (SK / 8), k = n % (SK / 8);
        const uint32_t row = raw + kshift + (k >> 1) * G::TILE + ((k & 1) * 8 + g) * KF::PITCH + (blk >> 1) * 2 * KF::BB;
        uint32_t f[4];
        if (KQ8) {
          const uint32_t w0 = blk & 1 ? lds32(row + 36 + 4 * t) : __byte_perm(lds32(row + 4 * t), lds32(row + 32), first_sel);
          unpack_q8(w0, &f[0], &f[1]);
          unpack_q8(lds32(row + (blk & 1 ? 52 : 16) + 4 * t), &f[2], &f[3]);
        } else {
          unpack_q4_subnormal(blk & 1 ? lds32(row + 20 + 4 * t) : __byte_perm(lds32(row + 4 * t), lds32(row + 16), first_sel), f);
        }
        *reinterpret_cast<uint4*>(smem + frag + n * 512) = make_uint4(f[0], f[1], f[2], f[3]);
      }
      // ---- V: the B operand of 16 keys x 32 dimensions
      for (int n = pwarp; n < NB * SUBS; n += PW) {
        const uint32_t blk = n / SUBS, j = n % SUBS;
        uint32_t f[4][2];
#pragma unroll
        for (int kp = 0; kp < 2; kp++) {
          const uint32_t row = raw + j * G::TILE + TK * KF::PITCH + vshift + (2 * t + 8 * kp) * VF::PITCH;
          if (VQ8) {
            uint32_t x[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const uint32_t pos = row + h * VF::PITCH + (blk >> 1) * 2 * VF::BB;
              x[h] = (blk & 1 ? lds32(pos + 36 + 4 * g) : __byte_perm(lds32(pos + 4 * g), lds32(pos + 32), first_sel_v)) ^ 0x80808080u;
            }
            const uint32_t lo2 = __byte_perm(x[0], x[1], 0x5140), hi2 = __byte_perm(x[0], x[1], 0x7362);
            f[0][kp] = h2_add(__byte_perm(lo2, 0x64646464u, 0x4140), 0xE480E480u);
            f[1][kp] = h2_add(__byte_perm(lo2, 0x64646464u, 0x4342), 0xE480E480u);
            f[2][kp] = h2_add(__byte_perm(hi2, 0x64646464u, 0x4140), 0xE480E480u);
            f[3][kp] = h2_add(__byte_perm(hi2, 0x64646464u, 0x4342), 0xE480E480u);
          } else {
            const uint32_t pos = row + blk * VF::BB + 2 + 2 * g;
            uint32_t x = __byte_perm(lds16(pos), lds16(pos + VF::PITCH), 0x5410);
            f[0][kp] = h2_add((x & 0x000F000Fu) | 0x64006400u, 0xE408E408u);
            f[1][kp] = h2_fma((x & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u);
            x >>= 8;
            f[2][kp] = h2_add((x & 0x000F000Fu) | 0x64006400u, 0xE408E408u);
            f[3][kp] = h2_fma((x & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u);
          }
        }
        *reinterpret_cast<uint4*>(smem + frag + G::KFRAG + n * 1024) = make_uint4(f[0][0], f[0][1], f[1][0], f[1][1]);
        *reinterpret_cast<uint4*>(smem + frag + G::KFRAG + n * 1024 + 512) = make_uint4(f[2][0], f[2][1], f[3][0], f[3][1]);
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(frag_full + 8 * buf);
      unpackers_sync();   // the raw stage has been read
      if (ptid == 0 && it + G::RAWS < stages) {
        issue(it + G::RAWS);
        place(it + G::RAWS + 1);
      }
    }
  } else {
  // ================ consumers ================
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CONSUMER_REGS));
  // ---- q as the A operand: rows g and g + 8, two terms, normed by the row's largest value to [2^13, 2^14)
  const uint32_t qf = G::OFF_QF + warp * ((D / 16) * 1024) + lane * 16;
  float factor[2];
  {
    float up[2] = {0.0f, 0.0f};
#pragma unroll 1
    for (int r = 0; r < 16; r++) {
      uint32_t l;
      const uint32_t row = row_of(warp * 16 + r, &l);
      float top = 0.0f;
      if (row != NO_ROW)
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
          const uint64_t at = (uint64_t)row * D + lane + 32 * i;
          top = fmaxf(top, fabsf(p.q_dtype == AION_CUDA_DTYPE_F32 ? static_cast<const float*>(p.q)[at] : __half2float(static_cast<const __half*>(p.q)[at])));
        }
      uint32_t e = __reduce_max_sync(FULL, __float_as_uint(top)) >> 23;
      if (e == 255) e = 127;
      e = max(e, 40u);
      if ((r & 7) == g) {
        const float to_base2 = p.soft_cap > 0.0f ? 1.0f : LOG2E;
        (r < 8 ? up[0] : up[1]) = __uint_as_float((127u + 13u + 127u - e) << 23);
        (r < 8 ? factor[0] : factor[1]) = p.scale * __uint_as_float((e - 13u) << 23) * to_base2;
      }
    }
#pragma unroll 1
    for (int blk = 0; blk < NB; blk++) {
      float part[2] = {0.0f, 0.0f};
#pragma unroll
      for (int m = 0; m < 2; m++) {
        uint32_t h4[4], l4[4];
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
          for (int half = 0; half < 2; half++) {   // operand order: (row g, r 0), (row g + 8, r 0), (row g, r 1), (row g + 8, r 1)
            float x[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const int dim = KQ8 ? pair_byte(true, blk & 1, t + 4 * m, 2 * r + h) : 2 * pair_byte(false, blk & 1, t, m + 2 * h) + r;
              x[h] = 0.0f;
              if (my_row[half] != NO_ROW) {
                const uint64_t at = (uint64_t)my_row[half] * D + blk * QK + dim;
                x[h] = p.q_dtype == AION_CUDA_DTYPE_F32 ? static_cast<const float*>(p.q)[at] : __half2float(static_cast<const __half*>(p.q)[at]);
              }
              x[h] = x[h] * up[half] * (!KQ8 && r ? 0.0625f : 1.0f);
            }
            split2(x[0], x[1], &h4[2 * r + half], &l4[2 * r + half]);
            if (!KQ8) {
              const float2 a = __half22float2(*reinterpret_cast<__half2*>(&h4[2 * r + half])), c = __half22float2(*reinterpret_cast<__half2*>(&l4[2 * r + half]));
              part[half] += ((a.x + c.x) + (a.y + c.y)) * (r ? 16.0f : 1.0f);
            }
          }
        *reinterpret_cast<uint4*>(smem + qf + (2 * blk + m) * 1024) = make_uint4(h4[0], h4[1], h4[2], h4[3]);
        *reinterpret_cast<uint4*>(smem + qf + (2 * blk + m) * 1024 + 512) = make_uint4(l4[0], l4[1], l4[2], l4[3]);
      }
      if (!KQ8) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
          part[half] += __shfl_xor_sync(FULL, part[half], 1);
          part[half] += __shfl_xor_sync(FULL, part[half], 2);
          if (t == 0) *reinterpret_cast<float*>(smem + G::OFF_CI + ((warp * NB + blk) * 16 + g + 8 * half) * 4) = part[half] * (-8.0f * 5.9604644775390625e-8f);
        }
      }
    }
  }
  __syncwarp();

#pragma unroll
  for (int i = 0; i < NB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) acc[i][j][e] = 0.0f;

  for (uint32_t it = 0; it < stages; it++) {
    const uint32_t buf = it & 1, frag = G::OFF_FRAG + buf * G::FRAG + lane * 16;
    if (!__all_sync(FULL, ptx::mbar_wait_bounded(frag_full + 8 * buf, (it >> 1) & 1, p.wait_limit))) {
      if (lane == 0) atomicExch(p.fault, FAULT_WAIT_EXPIRED), flags[1] = 1;
      break;
    }
    const uint32_t e_new = summary[buf].x, any_odd = summary[buf].y;
    // Does some row of this warp see a key of the stage, and do all of them see all?
    bool some = false, partial = false;
    uint32_t key0[SUBS], there[SUBS];
#pragma unroll
    for (int s = 0; s < SUBS; s++) {
      const uint2 v = valid[buf * SUBS + s];
      there[s] = v.x, key0[s] = v.y;
      some |= v.x && v.y < w_hi && v.y + TK > w_lo;
      partial |= v.x != 0xFFFFu || v.y < w_all_lo || v.y + TK > w_all_hi;
    }
    if (some) {

    // ---- S: rows g and g + 8, keys 8n + 2t and 8n + 2t + 1
    float s[SK / 8][4];
#pragma unroll
    for (int n = 0; n < SK / 8; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
    for (int blk = 0; blk < NB; blk++) {
      uint4 qh[2], ql[2];
#pragma unroll
      for (int m = 0; m < 2; m++) {
        qh[m] = *reinterpret_cast<const uint4*>(smem + qf + (2 * blk + m) * 1024);
        ql[m] = *reinterpret_cast<const uint4*>(smem + qf + (2 * blk + m) * 1024 + 512);
      }
      float ci[2] = {0.0f, 0.0f};
      if (!KQ8)
#pragma unroll
        for (int half = 0; half < 2; half++) ci[half] = *reinterpret_cast<const float*>(smem + G::OFF_CI + ((warp * NB + blk) * 16 + g + 8 * half) * 4);
      // (Step by step over all keys: neighbouring MMAs are independent.)
      uint4 f[SK / 8];
      float c[SK / 8][4];
#pragma unroll
      for (int n = 0; n < SK / 8; n++) {
        f[n] = *reinterpret_cast<const uint4*>(smem + frag + (blk * (SK / 8) + n) * 512);
        mma_f16_from(c[n], ql[0].x, ql[0].y, ql[0].z, ql[0].w, f[n].x, f[n].y, ci[0], ci[0], ci[1], ci[1]);
      }
#pragma unroll
      for (int n = 0; n < SK / 8; n++) mma_f16_from(c[n], ql[1].x, ql[1].y, ql[1].z, ql[1].w, f[n].z, f[n].w, c[n][0], c[n][1], c[n][2], c[n][3]);
#pragma unroll
      for (int n = 0; n < SK / 8; n++) mma_f16_from(c[n], qh[0].x, qh[0].y, qh[0].z, qh[0].w, f[n].x, f[n].y, c[n][0], c[n][1], c[n][2], c[n][3]);
#pragma unroll
      for (int n = 0; n < SK / 8; n++) mma_f16_from(c[n], qh[1].x, qh[1].y, qh[1].z, qh[1].w, f[n].z, f[n].w, c[n][0], c[n][1], c[n][2], c[n][3]);
#pragma unroll
      for (int n = 0; n < SK / 8; n++) {
        const float2 sc = lds_f2(G::OFF_KS + ((buf * NB + blk) * SK + 8 * n + 2 * t) * 4);
        s[n][0] = fmaf(sc.x, c[n][0], s[n][0]);
        s[n][1] = fmaf(sc.y, c[n][1], s[n][1]);
        s[n][2] = fmaf(sc.x, c[n][2], s[n][2]);
        s[n][3] = fmaf(sc.y, c[n][3], s[n][3]);
      }
    }
    // ---- softmax
    float m_new[2] = {m_run[0], m_run[1]}, unit[2] = {factor[0], factor[1]};
    if (!KQ8) {   // the codes' 2^24
#pragma unroll
      for (int n = 0; n < SK / 8; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[n][e] *= 16777216.0f;
    }
    if (p.soft_cap > 0.0f) {
#pragma unroll
      for (int n = 0; n < SK / 8; n++) {
#pragma unroll
        for (int e = 0; e < 4; e++) s[n][e] *= factor[e >> 1];
        cap_logits(s[n], p.soft_cap, 1.0f / p.soft_cap);
      }
      unit[0] = unit[1] = LOG2E;
    }
#pragma unroll
    for (int n = 0; n < SK / 8; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float y = s[n][e] * unit[e >> 1];
        if (partial) {
          const uint32_t k = (n & 1) * 8 + 2 * t + (e & 1), key = key0[n >> 1] + k;
          if (!((there[n >> 1] >> k) & 1) || key < lo[e >> 1] || key >= hi[e >> 1]) y = -INFINITY;
        }
        s[n][e] = y;
        m_new[e >> 1] = fmaxf(m_new[e >> 1], y);
      }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      m_new[h] = fmaxf(m_new[h], __shfl_xor_sync(FULL, m_new[h], 1));
      m_new[h] = fmaxf(m_new[h], __shfl_xor_sync(FULL, m_new[h], 2));
    }
    if (__any_sync(FULL, m_new[0] > m_run[0] || m_new[1] > m_run[1] || e_new > e_run)) {
      const float down = __uint_as_float((127u + e_run - e_new) << 23);
      float a[2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        a[h] = m_new[h] > m_run[h] ? ex2(m_run[h] - m_new[h]) : 1.0f;
        l_run[h] *= a[h];
        a[h] *= down;
        m_run[h] = m_new[h];
      }
      e_run = e_new;
#pragma unroll
      for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j][0] *= a[0], acc[i][j][1] *= a[0], acc[i][j][2] *= a[1], acc[i][j][3] *= a[1];
    }
    const float safe[2] = {m_run[0] == -INFINITY ? 0.0f : m_run[0], m_run[1] == -INFINITY ? 0.0f : m_run[1]};
#pragma unroll
    for (int n = 0; n < SK / 8; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[n][e] = ex2(s[n][e] - safe[e >> 1]);
        l_run[e >> 1] += s[n][e];
      }

    // ---- O += P' . V
#pragma unroll
    for (int blk = 0; blk < NB; blk++) {
      // (Summed from zero and added in f32: the tensor core cuts its sums off to one side.)
      float o[4][4];
#pragma unroll
      for (int i = 0; i < 4; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll
      for (int j = 0; j < SUBS; j++) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int kp = 0; kp < 2; kp++) {
          const float2 v = lds_f2(G::OFF_VS + ((buf * NB + blk) * SK + TK * j + 2 * t + 8 * kp) * 4);
          const float2 w0 = mul2(make_float2(s[2 * j + kp][0], s[2 * j + kp][1]), v), w1 = mul2(make_float2(s[2 * j + kp][2], s[2 * j + kp][3]), v);
          split2(w0.x, w0.y, &ah[2 * kp], &al[2 * kp]);
          split2(w1.x, w1.y, &ah[2 * kp + 1], &al[2 * kp + 1]);
        }
        const uint4 f0 = *reinterpret_cast<const uint4*>(smem + frag + G::KFRAG + (blk * SUBS + j) * 1024);
        const uint4 f1 = *reinterpret_cast<const uint4*>(smem + frag + G::KFRAG + (blk * SUBS + j) * 1024 + 512);
        const uint32_t bf[4][2] = {{f0.x, f0.y}, {f0.z, f0.w}, {f1.x, f1.y}, {f1.z, f1.w}};
#pragma unroll
        for (int i = 0; i < 4; i++) mma_f16_from(o[i], al[0], al[1], al[2], al[3], bf[i][0], bf[i][1], o[i][0], o[i][1], o[i][2], o[i][3]);
#pragma unroll
        for (int i = 0; i < 4; i++) mma_f16_from(o[i], ah[0], ah[1], ah[2], ah[3], bf[i][0], bf[i][1], o[i][0], o[i][1], o[i][2], o[i][3]);
      }
#pragma unroll
      for (int i = 0; i < 4; i++)
        add2(acc[blk][i][0], acc[blk][i][1], o[i][0], o[i][1]), add2(acc[blk][i][2], acc[blk][i][3], o[i][2], o[i][3]);
    }
    if (any_odd) {   // a V scale that is not finite: NaN where a row gives weight to its key
#pragma unroll
      for (int blk = 0; blk < NB; blk++) {
        const uint32_t which = odd[buf * NB + blk];
        bool met[2] = {false, false};
#pragma unroll
        for (int n = 0; n < SK / 8; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) met[e >> 1] |= ((which >> (8 * n + 2 * t + (e & 1))) & 1) && s[n][e] > 0.0f;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const uint32_t who = __ballot_sync(FULL, met[h]);
          const float add = (who >> (4 * g)) & 15 ? NAN : 0.0f;
#pragma unroll
          for (int i = 0; i < 4; i++) acc[blk][i][2 * h] += add, acc[blk][i][2 * h + 1] += add;
        }
      }
    }
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(frag_empty + 8 * buf);   // the fragments have been read
  }

  // ---- the rows' sums: straight out, or through shared memory to the cluster's others
#pragma unroll
  for (int h = 0; h < 2; h++) {
    l_run[h] += __shfl_xor_sync(FULL, l_run[h], 1);
    l_run[h] += __shfl_xor_sync(FULL, l_run[h], 2);
  }
  const float back = __uint_as_float((127u + e_run - 29u) << 23);
  const bool report = !flags[0] && !flags[1];
  float* res = reinterpret_cast<float*>(smem + G::OFF_QF);
  float* stats = reinterpret_cast<float*>(smem + G::OFF_STATS);
  __syncwarp();   // (a warp's sums take the place of its own queries)
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const uint32_t r = warp * 16 + g + 8 * h;
    const bool good = l_run[h] > 0.0f && isfinite(l_run[h]);
    float mul = back;
    float* dst = res + r * D;
    if (rg.cluster == 1) {
      if (my_row[h] == NO_ROW) continue;
      if (!good && hi[h] > lo[h] && report) atomicCAS(p.fault, FAULT_NONE, FAULT_NONFINITE);
      mul = good ? back * __frcp_rn(l_run[h]) : 0.0f;
      dst = p.out + (uint64_t)my_row[h] * D;
    } else if (t == 0) {
      stats[r] = m_run[h], stats[ROWS + r] = l_run[h];
    }
#pragma unroll
    for (int blk = 0; blk < NB; blk++)
#pragma unroll
      for (int c = 0; c < 2; c++) {   // dimensions of the column group 2t + c
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = rg.cluster == 1 && !good ? 0.0f : acc[blk][i][2 * h + c] * mul;
        float* at = dst + blk * QK;
        if (VQ8) {
          const int d0 = pair_byte(true, blk & 1, 2 * t + c, 0), d2 = pair_byte(true, blk & 1, 2 * t + c, 2);
          *reinterpret_cast<float2*>(at + d0) = make_float2(v[0], v[1]);
          *reinterpret_cast<float2*>(at + d2) = make_float2(v[2], v[3]);
        } else {
          *reinterpret_cast<float4*>(at + 4 * (2 * t + c)) = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
  }
  }   // consumers
  if (rg.cluster == 1) return;
  const bool report = !flags[0] && !flags[1];
  cluster_sync();
  const uint32_t share = ROWS / rg.cluster, res_addr = sbase + G::OFF_QF, stats_addr = sbase + G::OFF_STATS;
  for (uint32_t i = tid; i < share * (D / 4); i += RTHREADS) {
    const uint32_t r = rank * share + i / (D / 4), d4 = i % (D / 4);
    uint32_t l;
    const uint32_t row = row_of(r, &l);
    if (row == NO_ROW) continue;
    float m[8], w[8], M = -INFINITY, lsum = 0.0f;
    float4 v[8], o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < 8; k++) {
      m[k] = -INFINITY, w[k] = 0.0f, v[k] = o;
      if (k < (int)rg.cluster) {
        const uint32_t a = cluster_addr(stats_addr, k);
        m[k] = ld_cluster_f(a + 4 * r), w[k] = ld_cluster_f(a + 4 * (ROWS + r));
        v[k] = ld_cluster_f4(cluster_addr(res_addr, k) + (r * D + 4 * d4) * 4);
      }
      M = fmaxf(M, m[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float f = m[k] == -INFINITY ? 0.0f : ex2(m[k] - M);
      o.x += v[k].x * f, o.y += v[k].y * f, o.z += v[k].z * f, o.w += v[k].w * f;
      lsum += w[k] * f;
    }
    const bool good = lsum > 0.0f && isfinite(lsum);
    if (!good && d4 == 0 && report) {
      const KeyRange kr = key_range(p, b, l);
      if (kr.hi > kr.lo) atomicCAS(p.fault, FAULT_NONE, FAULT_NONFINITE);
    }
    const float inv = good ? __frcp_rn(lsum) : 0.0f;
    *reinterpret_cast<float4*>(p.out + (uint64_t)row * D + 4 * d4) = good ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  cluster_sync();   // no CTA leaves before the others have read its sums
}

template <int D, bool KQ8, bool VQ8>
int32_t launch_rows(AionCudaDevice* dev, const AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, uint64_t max_keys) {
  using G = RowsGeom<D, KQ8, VQ8>;
  auto kernel = attn_qcache_rows_kernel<D, KQ8, VQ8>;
  // Clusters of 1, 2, 4 and 8 CTAs that the device holds at once; worked out once per device and instantiation.
  uint32_t held[4];
  {
    static std::mutex mu;
    static uint32_t known[64][4] = {};
    std::lock_guard<std::mutex> lock(mu);
    if (dev->ordinal < 0 || dev->ordinal >= 64) return fail(AION_CUDA_UNSUPPORTED, "attention: device %d", dev->ordinal);
    if (!known[dev->ordinal][0]) {
      AION_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM));
      prefer_max_shared(reinterpret_cast<const void*>(kernel));
      for (int i = 3; i >= 0; i--) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(8);
        cfg.blockDim = dim3(RTHREADS);
        cfg.dynamicSmemBytes = G::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1u << i, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        AION_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
        known[dev->ordinal][i] = n > 0 ? (uint32_t)n : 1u;
      }
    }
    for (int i = 0; i < 4; i++) held[i] = known[dev->ordinal][i];
  }
  RowsGrid rg{};
  rg.rows = p.L * (p.Hq / p.Hkv);
  rg.row_blocks = (rg.rows + ROWS - 1) / ROWS;
  const uint64_t units = (uint64_t)p.B * rg.row_blocks * p.Hkv;
  // One CTA an SM. The keys are cut over as many CTAs as finish soonest in rounds of what the device holds at once
  // (clusters of eight fit only where a group of SMs has as many free), four stages each at least; a cluster's sums
  // cost about as much as eight stages.
  rg.cluster = 1;
  double best = 1e30;
  for (uint32_t c = 1, i = 0; c <= 8 && max_keys >= (uint64_t)c * (c > 1 ? 4 : 0) * SK; c *= 2, i++) {
    const double cost = std::ceil((double)units / held[i]) * (std::ceil((double)max_keys / (c * SK)) + 4.0 + (c > 1 ? 8.0 : 0.0));
    if (cost < best) best = cost, rg.cluster = c;
  }
  if (units * rg.cluster > 0x7FFFFFFFull) return fail(AION_CUDA_UNSUPPORTED, "attention: too many rows");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * rg.cluster));
  cfg.blockDim = dim3(RTHREADS);
  cfg.dynamicSmemBytes = G::SMEM;
  cfg.stream = dev->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = rg.cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  static const bool no_pdl_main = std::getenv("AION_CUDA_NO_PDL_MAIN") != nullptr;  // tuning only
  cfg.numAttrs = no_pdl_main ? 1 : 2;
  AION_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p, rg, tk, tv));
  return AION_CUDA_OK;
}

}  // namespace

int32_t attention_qcache_rows(AionCudaDevice* dev, const AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, uint64_t max_keys) {
  const bool kq8 = p.k_dtype == AION_CUDA_DTYPE_Q8_0, vq8 = p.v_dtype == AION_CUDA_DTYPE_Q8_0;
#define AION_QROWS(D)                                                                                                                  \
  if (kq8) return vq8 ? launch_rows<D, true, true>(dev, p, tk, tv, max_keys) : launch_rows<D, true, false>(dev, p, tk, tv, max_keys); \
  return vq8 ? launch_rows<D, false, true>(dev, p, tk, tv, max_keys) : launch_rows<D, false, false>(dev, p, tk, tv, max_keys);
  switch (p.Dk) {
    case 64: AION_QROWS(64)
    case 128: AION_QROWS(128)
    default: AION_QROWS(256)
  }
#undef AION_QROWS
}

}  // namespace aion
