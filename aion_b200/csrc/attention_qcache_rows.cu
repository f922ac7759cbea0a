// `Attention` over a quantized KV cache for many query rows (prompts, several new rows per request): a CTA holds up to 128
// rows of one kv head, a row being (query position, query head of the group), and streams the keys once for all of them,
// 64 to a stage, through the tensor cores of the fifth generation.
//
//  * f32 attention on f16 operands: q, P = exp2(S - max), and the dequantized K and V (code * scale is 19 bits) are two f16
//    terms each, and each product is the sum of three (lo.hi, hi.lo, hi.hi; what is left out is 2^-22). So the tensor pipe does
//    6 * 2 * rows * keys * D operations for the 4 * rows * keys * D that f32 attention counts: a third of its rate is the ceiling.
//    P's second term is held times 2^11 and scaled back as the sum goes on (scale-input-d): the power of two that P is normed by
//    follows the largest V scale that any row of the block sees, and so a weight on a small V keeps its 23 bits down to 2^-28 of it.
//  * A row of a cache is brought to a common power of two, so that its largest scale lies in [2^14, 2^15), and its codes count
//    1/128 each: a scale next to a larger one of its row is exact over 28 powers of two, and one next to another row's
//    loses nothing at all. Code times scale is exact down to 2^-21 of the row's largest scale, below that good to 2^-32 of
//    it. The power comes back per key, times the logit and times P.
//  * Both products take A from tensor memory: q (two terms, D columns) stays there for the whole walk, P overwrites the logits
//    it is made of. Shared memory holds the two B operands, one 128-byte-swizzled panel per 64 dimensions, K read K-major and V
//    N-major, so that both are unpacked the same way.
//  * O of a stage is summed from zero in tensor memory, 64 dimensions at a time in two buffers, and added in f32 registers (the
//    tensor core cuts its sums off to one side; and the running maximum then costs no trip to tensor memory and back).
//  * Eight warps do the softmax and hold O (a thread: one row, half of the keys and of every 64 dimensions), six unpack, one
//    issues the products, one the TMA boxes of 16 rows. The product of the next stage's logits is issued before this stage's
//    P . V, so that the softmax runs under it.
//  * A context too long for the few CTAs of a short prompt is cut over a cluster, whose CTAs add up their sums through
//    distributed shared memory.
//
// 1024 rows against 8192 keys, 8 heads over 4 kv heads of 256, q8_0: 224 us, 288 TFLOP/s of the 4 * rows * keys * D that attention
// counts (the products alone take 118 us at 1634 TFLOP/s); a causal prompt of 4096 tokens 218 us, 315 TFLOP/s; 32 over 8
// heads of 128 552 us, 233 TFLOP/s. (On m16n8k16, eight warps of sixteen rows that held all in registers: 616, 596 and 1129 us.)
// What bounds it: the hand-overs between the roles of a stage; the tensor pipe is active 48 % of the cycles (59 % on the busiest
// SM). The loop is straight code of four kinds and has to fit the instruction cache: with the products spelled out (their
// descriptors went to local memory), a report in every wait and the unpacking once per block and operand it took 378 us.
#include <cmath>
#include <cstdlib>
#include <mutex>

#include "attention_qcache.cuh"
#include "tcgen05.cuh"

namespace aion {

namespace {

using namespace qcache;

constexpr int CW = 8;                 // softmax warps
constexpr int MMA_WARP = 8, LOAD_WARP = 9, FIRST_UNPACK = 10;
constexpr int UW = 6;                 // unpacking warps
constexpr int RTHREADS = 16 * 32;
constexpr int ROWS = 128;
constexpr int SUBS = 4;               // tiles of a stage
constexpr int SK = SUBS * TK;         // keys of a stage
constexpr int KRAWS = 3, VRAWS = 2;   // raw stages
constexpr int SLOTS = 4;              // stages whose exponents and masks are kept
// Registers of a softmax warp's thread and of the others'; they add up to what the block is launched with, 128 each. (Heads of
// 256, whose sums alone take 128, were 2 % slower with 192 and 64, heads of 128 3 % faster.)
constexpr int softmax_regs(int d) { return d == 256 ? 200 : 192; }
constexpr int other_regs(int d) { return 256 - softmax_regs(d); }
static_assert(SK == 64 && FIRST_UNPACK + UW == RTHREADS / 32, "a stage is one panel of 64 keys");
constexpr int PANEL = SK * 128;       // bytes of 64 keys x 64 dimensions of f16

struct RowsGrid {
  uint32_t cluster;      // CTAs that share a unit's keys
  uint32_t row_blocks;   // blocks of ROWS rows per (request, kv head)
  uint32_t rows;         // L * query heads of the group
};

template <int D, bool KQ8, bool VQ8>
struct RowsGeom {
  using K = RowFmt<D, KQ8>;
  using V = RowFmt<D, VQ8>;
  static constexpr int NP = D / 64;
  static constexpr int KRAW = SK * K::PITCH, VRAW = SK * V::PITCH;
  static constexpr int OFF_K = 0;                                // [hi, lo][panel]; first f32 q [ROWS][D], at the end f32 sums
  static constexpr int OFF_V = OFF_K + 2 * NP * PANEL;           // [hi, lo][panel]
  static constexpr int OFF_KRAW = OFF_V + 2 * NP * PANEL;
  static constexpr int OFF_VRAW = OFF_KRAW + KRAWS * KRAW;
  static constexpr int OFF_KEXP = OFF_VRAW + VRAWS * VRAW;       // f32 [SLOTS][SK]: the keys' powers of two
  static constexpr int OFF_VEXP = OFF_KEXP + SLOTS * SK * 4;
  static constexpr int OFF_KSC = OFF_VEXP + SLOTS * SK * 4;      // f16 [2][SK][blocks]: the scales, normed
  static constexpr int OFF_VSC = OFF_KSC + 2 * SK * NP * 4;      // f16 [3][SK][blocks]
  static constexpr int OFF_EX = OFF_VSC + 3 * SK * NP * 4;       // f32 [2][2][ROWS]: maxima (or NaN blocks) of the two halves of a row
  static constexpr int OFF_STATS = OFF_EX + 4 * ROWS * 4;        // f32 [2][ROWS]: the rows' maxima and weights, for the cluster
  static constexpr int OFF_ROWS = OFF_STATS + 2 * ROWS * 4;      // u32 [ROWS]: a row's place in q and out
  static constexpr int OFF_VMAX = OFF_ROWS + ROWS * 4;      // u32 [SLOTS][8]: largest V exponent that an unpacking warp met, 256 for a scale that is not finite
  static constexpr int OFF_VALID = OFF_VMAX + SLOTS * 8 * 4;     // uint2 [SLOTS][SUBS]: which keys are there, the first of them
  static constexpr int OFF_ODD = OFF_VALID + SLOTS * SUBS * 8;   // u8 [SLOTS][SK]: blocks of a key whose V scale is not finite
  static constexpr int OFF_PAIR = OFF_ODD + SLOTS * SK;          // u32 [2][2][4]: did the half of the rows meet such a scale?
  static constexpr int OFF_BARS = OFF_PAIR + 16 * 4;
  static constexpr int OFF_FLAGS = OFF_BARS + 28 * 8;             // bad inputs, gave up, TMEM, -, first key, key end
  static constexpr int SMEM = OFF_FLAGS + 32 + 1024;             // (panels begin on 1024 bytes)
  static_assert(4 * NP * PANEL == ROWS * D * 4 && OFF_KRAW % 128 == 0 && KRAW % 128 == 0 && VRAW % 128 == 0 && SMEM <= 227 * 1024, "shared memory");
  // tensor memory: columns of 32 bits
  static constexpr uint32_t T_Q = 0, T_S = D, T_O = D + 2 * 64;
  static_assert(T_O + 2 * 64 <= 512, "tensor memory");
};

// D f32, A and B f16, M = 128, N = 64; B K-major, or (bit 16) N-major.
constexpr uint32_t IDESC_QK = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24), IDESC_PV = IDESC_QK | (1u << 16);

// D[tmem] (+)= A[tmem] . B[smem desc], four steps of K = 16: A eight columns further each (the third and fourth SKIP more), B
// STEP units of its descriptor. The whole warp comes here and one elected thread, always the same, issues: so the operands stay
// in uniform registers and an instruction is issued in the 32 clocks that it takes. (Inside a branch of one thread 49 clocks each.)
// What D holds before is worth 2^-DOWN of it.
template <int SKIP, int STEP, int DOWN = 0>
__device__ __forceinline__ void umma_f16_ts4(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b32 a1, a2, a3;\n\telect.sync _|e, 0xFFFFFFFF;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "add.u32 a1, %1, 8;\n\tadd.u32 a2, %1, %5;\n\tadd.u32 a3, %1, %6;\n\tadd.u64 b1, %2, %7;\n\tadd.u64 b2, %2, %8;\n\tadd.u64 b3, %2, %9;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, %10;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, 1;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, 1;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate), "n"(16 + SKIP), "n"(24 + SKIP), "n"(STEP), "n"(2 * STEP), "n"(3 * STEP), "n"(DOWN)
      : "memory");
}
__device__ __forceinline__ void umma_commit_elected(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xFFFFFFFF;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32f(uint32_t taddr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
      "%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
        "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]),
        "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]),
        "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
      "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16f(uint32_t taddr, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
        "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(CW * 32) : "memory"); }
__device__ __forceinline__ void unpack_sync() { asm volatile("bar.sync 6, %0;" ::"n"(UW * 32) : "memory"); }
// The two warps that hold the halves of the same 32 rows.
__device__ __forceinline__ void pair_sync(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(2 + quarter) : "memory"); }
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_rest(uint32_t a, uint32_t b, uint32_t c) {   // a * b - c
  const __half2 d = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b), __hneg2(*reinterpret_cast<__half2*>(&c)));
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The panels of a stage: lanes are 32 / NP keys x NP panels of 64 dimensions (two blocks), the warps share key groups and
// the two blocks of a panel.
template <int D, bool Q8>
struct Unpack {
  using F = RowFmt<D, Q8>;
  static constexpr int NP = D / 64, KPW = 32 / NP, GROUPS = SK / KPW;
  // Scales of the key's two blocks in this lane's panel and the key's exponent: the largest of its finite scales'.
  static __device__ __forceinline__ uint32_t scales(const uint8_t* row, uint32_t (&sc)[2]) {
    sc[0] = *reinterpret_cast<const uint16_t*>(row);
    sc[1] = *reinterpret_cast<const uint16_t*>(row + F::BB);
    uint32_t e = 1;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const uint32_t x = (sc[i] >> 10) & 31;
      e = x < 31 ? max(e, x) : e;
    }
#pragma unroll
    for (int x = KPW; x < 32; x *= 2) e = max(e, __shfl_xor_sync(FULL, e, x));
    return e;
  }
  // The two scales in units of 2^(e - 29).
  static __device__ __forceinline__ uint32_t normed(const uint32_t (&sc)[2], uint32_t e) {
    const float up = pow2f(29 - (int)e);
    return pack_half2(half_bits(sc[0]) * up, half_bits(sc[1]) * up);
  }
  // One block of a key (the panel's first or second): 32 codes, 1/128 each, times its (normed) scale, as two f16 terms. `row` is where the
  // panel's bytes begin. (One code for both: the loop's instructions have to stay in the cache, see the kernel.)
  static __device__ __forceinline__ void block(const uint8_t* row, uint32_t second, uint32_t pair, uint8_t* hi, uint8_t* lo, uint32_t key) {
    const uint32_t s2 = __byte_perm(pair, 0, second ? 0x3232 : 0x1010);
    constexpr int CODES = Q8 ? 8 : 4;   // words of codes; the second block's begin in the middle of the word before
    uint32_t w[CODES];
    {
      const uint32_t* words = reinterpret_cast<const uint32_t*>(row) + (second ? CODES : 0);
      const uint32_t sel = second ? 0x7654 : 0x5432;
      uint32_t raw[CODES + 1];
#pragma unroll
      for (int i = 0; i <= CODES; i++) raw[i] = words[i];
#pragma unroll
      for (int i = 0; i < CODES; i++) w[i] = __byte_perm(raw[i], raw[i + 1], sel);
    }
    const uint32_t first = (second * 4) ^ (key & 7);
    auto store = [&](int c, const uint32_t (&u)[4]) {   // eight dimensions
      uint32_t h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        h[i] = h2_mul(u[i], s2);
        l[i] = h2_rest(u[i], s2, h[i]);   // exact: what the rounding left
      }
      const uint32_t at = key * 128 + ((first ^ c) << 4);
      *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
    };
    if (Q8) {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {   // 0x6400 | (n + 128) is 1152 + n: 9 + n / 128
          const uint32_t x = w[2 * c + i] ^ 0x80808080u;
          u[2 * i] = h2_fma(__byte_perm(x, 0x64646464u, 0x4140), 0x20002000u, 0xC880C880u);
          u[2 * i + 1] = h2_fma(__byte_perm(x, 0x64646464u, 0x4342), 0x20002000u, 0xC880C880u);
        }
        store(c, u);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++)   // a byte's low and high nibble, 1024 + n and 1024 + 16 n: 8 + n / 128 and 1/2 + n / 128
          u[i] = h2_fma((__byte_perm(w[c], 0, 0x4040 + 0x0101 * i) & 0x00F0000Fu) | 0x64006400u, 0x10002000u, 0xB880C808u);
        store(c, u);
      }
    }
  }
};

template <int D, bool KQ8, bool VQ8, bool CAP>
__global__ void __launch_bounds__(RTHREADS, 1) attn_qcache_rows_kernel(const AttnParams p, const RowsGrid rg, const __grid_constant__ CUtensorMap tmap_k,
                                                                      const __grid_constant__ CUtensorMap tmap_v) {
  using G = RowsGeom<D, KQ8, VQ8>;
  using KF = RowFmt<D, KQ8>;
  using VF = RowFmt<D, VQ8>;
  constexpr int NP = G::NP;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sbase = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - ptx::smem_u32(smem_raw));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bars = sbase + G::OFF_BARS;
  const uint32_t kraw_full = bars, kraw_empty = bars + 24, vraw_full = bars + 48, vraw_empty = bars + 64;   // [3], [3], [2], [2]
  const uint32_t k_ready = bars + 80, k_free = bars + 88, v_free = bars + 96, q_ready = bars + 104, done = bars + 112;
  const uint32_t s_full = bars + 120, p_ready = bars + 136, o_full = bars + 152, o_free = bars + 168, scaled = bars + 184;   // [2] x 4, [SLOTS]
  volatile uint32_t* flags = reinterpret_cast<uint32_t*>(smem + G::OFF_FLAGS);
  uint2* valid = reinterpret_cast<uint2*>(smem + G::OFF_VALID);
  const bool softmax = warp < CW;

  if (tid == 0) {
    for (int s = 0; s < KRAWS; s++) ptx::mbar_init(kraw_full + 8 * s, 1), ptx::mbar_init(kraw_empty + 8 * s, UW);
    for (int s = 0; s < 2; s++) {
      ptx::mbar_init(vraw_full + 8 * s, 1), ptx::mbar_init(vraw_empty + 8 * s, UW);
      ptx::mbar_init(s_full + 8 * s, 1), ptx::mbar_init(p_ready + 8 * s, CW + UW);
      ptx::mbar_init(o_full + 8 * s, 1), ptx::mbar_init(o_free + 8 * s, CW);
    }
    for (int s = 0; s < SLOTS; s++) ptx::mbar_init(scaled + 8 * s, UW);
    ptx::mbar_init(k_ready, UW), ptx::mbar_init(k_free, 1), ptx::mbar_init(v_free, 1);
    ptx::mbar_init(q_ready, CW), ptx::mbar_init(done, 1);
    flags[0] = flags[1] = flags[5] = 0;
    flags[4] = 0xFFFFFFFFu;
    ptx::fence_barrier_init();
  }
  for (int i = tid; i < SLOTS * 8; i += RTHREADS) *reinterpret_cast<uint32_t*>(smem + G::OFF_VMAX + 4 * i) = 0;
  if (warp == MMA_WARP) {
    tmem_alloc(sbase + G::OFF_FLAGS + 8, 512);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = flags[2];
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
  const int quarter = warp & 3, half = (warp >> 2) & 1;   // of a softmax warp: its 32 rows, its half of the keys and dimensions
  const uint32_t r = quarter * 32 + lane;
  uint32_t* rows = reinterpret_cast<uint32_t*>(smem + G::OFF_ROWS);
  uint32_t my_row = NO_ROW, lo = 0, hi = 0, all_lo = 0, all_hi = 0xFFFFFFFFu;
  if (softmax) {
    uint32_t l;
    my_row = row_of(r, &l);
    if (half == 0) rows[r] = my_row;
    if (my_row != NO_ROW) {
      const KeyRange kr = key_range(p, b, l);
      if (kr.bad) flags[0] = 1;
      lo = all_lo = kr.lo, hi = all_hi = kr.hi;
    }
    const uint32_t first = __reduce_min_sync(FULL, hi > lo ? lo : 0xFFFFFFFFu), last = __reduce_max_sync(FULL, hi > lo ? hi : 0u);
    all_lo = __reduce_max_sync(FULL, all_lo), all_hi = __reduce_min_sync(FULL, all_hi);   // what all rows of the warp see
    if (lane == 0 && last > 0) atomicMin(const_cast<uint32_t*>(flags) + 4, first), atomicMax(const_cast<uint32_t*>(flags) + 5, last);
  }
  __syncthreads();
  if (flags[0] && tid == 0) atomicExch(p.fault, FAULT_INVALID_ARGUMENT);
  const uint32_t u_hi = flags[5], u_lo = min(flags[4], u_hi);
  const TileSpace ts = tile_space(geom_of(p));
  const TileRange whole = tiles_of_keys(ts, u_lo, u_hi);
  uint32_t per = (whole.end - whole.first + rg.cluster - 1) / rg.cluster;
  per = (per + SUBS - 1) / SUBS * SUBS;
  const uint32_t my_first = (uint32_t)min((uint64_t)whole.end, whole.first + (uint64_t)rank * per);
  const uint32_t tiles = min(whole.end - my_first, per), stages = (tiles + SUBS - 1) / SUBS;

  // A wait that runs out is reported at the end; the warp then walks on without waiting or working, so that every arrival still comes and
  // no warp is left at a barrier of a pair.
  bool dead = false;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; !dead && !__all_sync(FULL, ptx::mbar_try_wait_spin(bar, parity & 1)); i++) dead = (i >> 4) >= p.wait_limit;   // (short polls)
  };
  auto report_wait = [&]() {
    if (dead && lane == 0) atomicExch(p.fault, FAULT_WAIT_EXPIRED), flags[1] = 1;
  };
  auto arrive = [&](uint32_t bar) {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar);
  };

  if (softmax) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(softmax_regs(D)));
    float factor;
    // ---- q into tensor memory: rows whole through shared memory, then normed by their largest value to [2^13, 2^14) and split
    {
      float* stage = reinterpret_cast<float*>(smem + G::OFF_K);
      float* tops = reinterpret_cast<float*>(smem + G::OFF_STATS);
#pragma unroll 1
      for (int i0 = 0; i0 < ROWS / CW; i0 += 8) {   // (eight rows' loads at once)
        float x[8][D / 32];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const uint32_t row = rows[warp * (ROWS / CW) + i0 + i];
          const uint64_t at = (uint64_t)row * D + lane;
          if (row == NO_ROW) {
#pragma unroll
            for (int j = 0; j < D / 32; j++) x[i][j] = 0.0f;
          } else if (p.q_dtype == AION_CUDA_DTYPE_F32) {
#pragma unroll
            for (int j = 0; j < D / 32; j++) x[i][j] = __ldg(static_cast<const float*>(p.q) + at + 32 * j);
          } else {
#pragma unroll
            for (int j = 0; j < D / 32; j++) x[i][j] = __half2float(__ldg(static_cast<const __half*>(p.q) + at + 32 * j));
          }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const uint32_t row_in = warp * (ROWS / CW) + i0 + i;
          float top = 0.0f;
#pragma unroll
          for (int j = 0; j < D / 32; j++) {
            const uint32_t d = lane + 32 * j;
            top = fmaxf(top, fabsf(x[i][j]));
            stage[row_in * D + ((((d >> 2) ^ (row_in & 7)) << 2) | (d & 3))] = x[i][j];
          }
          const uint32_t t = __reduce_max_sync(FULL, __float_as_uint(top));
          if (lane == 0) tops[row_in] = __uint_as_float(t);
        }
      }
      softmax_sync();
      uint32_t e = __float_as_uint(tops[r]) >> 23;
      if (e == 255) e = 127;
      e = max(e, 40u);
      const float up = __uint_as_float((127u + 13u + 127u - e) << 23);
      factor = p.scale * __uint_as_float((e - 13u) << 23) * (CAP ? 1.0f : LOG2E);
      const uint32_t tq = tmem + ((uint32_t)quarter << 21) + G::T_Q + half * (D / 4);
#pragma unroll 1
      for (int c = 0; c < D / 64; c++) {   // 32 dimensions
        uint32_t h[16], l[16];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const uint32_t chunk = half * (D / 8) + c * 8 + i;
          const float4 x = *reinterpret_cast<const float4*>(stage + r * D + ((chunk ^ (r & 7)) << 2));
          split2(x.x * up, x.y * up, &h[2 * i], &l[2 * i]);
          split2(x.z * up, x.w * up, &h[2 * i + 1], &l[2 * i + 1]);
        }
        tmem_st16(tq + c * 16, h);
        tmem_st16(tq + D / 2 + c * 16, l);
      }
      tmem_st_wait();
      tc_fence_before();
      arrive(q_ready);
    }
    float acc[NP][32];
#pragma unroll
    for (int q = 0; q < NP; q++)
#pragma unroll
      for (int i = 0; i < 32; i++) acc[q][i] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;
    uint32_t e_run = 0;
    float* ex = reinterpret_cast<float*>(smem + G::OFF_EX);
    const uint32_t lane_base = tmem + ((uint32_t)quarter << 21) + half * 32;

    // O of a stage, 64 dimensions: the other half of the warps takes the other 32.
    float a_of = 1.0f;   // what the sums so far are worth in units of that stage
    auto drain = [&](uint32_t it, int q, float (&sums)[32]) {
      const uint32_t n = it * NP + q;
      wait(o_full + 8 * (n & 1), n >> 1);
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < 2; j++) {
        float o[16];
        tmem_ld16f(lane_base + G::T_O + (n & 1) * 64 + j * 16, o);
        tmem_ld_wait();
        if (j == 1) {
          tc_fence_before();
          arrive(o_free + 8 * (n & 1));
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float2 x = fma2(make_float2(sums[16 * j + 2 * i], sums[16 * j + 2 * i + 1]), make_float2(a_of, a_of), make_float2(o[2 * i], o[2 * i + 1]));
          sums[16 * j + 2 * i] = x.x, sums[16 * j + 2 * i + 1] = x.y;
        }
      }
    };
    // P of stage `it`, in four steps, and between them O of the stage before, panel by panel as it comes.
    for (uint32_t it = 0; it <= stages; it++) {
      const bool more = it < stages, prev = it > 0;
      const uint32_t slot = it % SLOTS, at = lane_base + G::T_S + (it & 1) * 64;
      float s[32];
      float a_next = 1.0f;
      float* mx = ex + (it & 1) * 2 * ROWS;
      uint32_t any_odd = 0;
      if (more) {   // logits, the running maximum
        wait(scaled + 8 * slot, it / SLOTS);
        wait(s_full + 8 * (it & 1), it >> 1);
        tc_fence_after();
        tmem_ld32f(at, s);
        const uint4 v0 = *reinterpret_cast<const uint4*>(smem + G::OFF_VMAX + slot * 32), v1 = *reinterpret_cast<const uint4*>(smem + G::OFF_VMAX + slot * 32 + 16);
        const uint32_t met = max(max(v0.x & 31, v0.y & 31), max(max(v0.z & 31, v0.w & 31), max(v1.x & 31, v1.y & 31)));
        const uint32_t e_new = max(e_run, met);
        any_odd = (v0.x | v0.y | v0.z | v0.w | v1.x | v1.y) & 256;
        bool partial = false;
        uint32_t there[2], key0[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint2 v = valid[slot * SUBS + 2 * half + j];
          there[j] = v.x, key0[j] = v.y;
          partial |= v.x != 0xFFFFu || v.y < all_lo || v.y + TK > all_hi;
        }
        const float4* kexp = reinterpret_cast<const float4*>(smem + G::OFF_KEXP + (slot * SK + half * 32) * 4);
        tmem_ld_wait();
        if (CAP) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float4 k = kexp[i];
            float x[4] = {s[4 * i] * k.x * factor, s[4 * i + 1] * k.y * factor, s[4 * i + 2] * k.z * factor, s[4 * i + 3] * k.w * factor};
            cap_logits(x, p.soft_cap, inverse_cap(p.soft_cap));
#pragma unroll
            for (int j = 0; j < 4; j++) s[4 * i + j] = x[j] * LOG2E;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const float4 k = kexp[i];
            const float2 a = mul2(mul2(make_float2(s[4 * i], s[4 * i + 1]), make_float2(k.x, k.y)), make_float2(factor, factor));
            const float2 c = mul2(mul2(make_float2(s[4 * i + 2], s[4 * i + 3]), make_float2(k.z, k.w)), make_float2(factor, factor));
            s[4 * i] = a.x, s[4 * i + 1] = a.y, s[4 * i + 2] = c.x, s[4 * i + 3] = c.y;
          }
        }
        if (partial) {
#pragma unroll
          for (int i = 0; i < 32; i++) {
            const uint32_t key = key0[i >> 4] + (i & 15);
            if (!((there[i >> 4] >> (i & 15)) & 1) || key < lo || key >= hi) s[i] = -INFINITY;
          }
        }
        float top[4] = {m_run, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; i++) top[i & 3] = fmaxf(top[i & 3], s[i]);
        const float mine = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        uint32_t* both = reinterpret_cast<uint32_t*>(smem + G::OFF_PAIR) + (it & 1) * 8 + quarter;
        mx[half * ROWS + r] = mine;
        if (lane == 0) both[4 * half] = any_odd;
        pair_sync(quarter);
        any_odd = both[0] | both[4];   // (the two warps go the same way, even when one of them has given up waiting)
        const float m_new = fmaxf(mine, mx[(half ^ 1) * ROWS + r]);
        const float a = m_new > m_run ? ex2(m_run - m_new) : 1.0f;
        l_run *= a;
        a_next = a * pow2f((int)e_run - (int)e_new);
        m_run = m_new, e_run = e_new;
      }
      if (prev) {
        drain(it - 1, 0, acc[0]);
        if (NP > 1) drain(it - 1, 1, acc[1 % NP]);
      }
      if (more) {   // weights
        const float off = m_run == -INFINITY ? 0.0f : -m_run;
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int i = 0; i < 16; i++) {
          float2 x = make_float2(s[2 * i], s[2 * i + 1]);
          add2(x.x, x.y, off, off);
          x.x = ex2(x.x), x.y = ex2(x.y);
          add2(sum[i & 1].x, sum[i & 1].y, x.x, x.y);
          s[2 * i] = x.x, s[2 * i + 1] = x.y;
        }
        l_run += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      if (any_odd) {   // a V scale that is not finite: NaN where a row gives weight to its key
        const uint8_t* odd = smem + G::OFF_ODD + slot * SK + half * 32;
        uint32_t hit = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) hit |= s[i] > 0.0f ? odd[i] : 0u;
        pair_sync(quarter);   // (the maxima have been read)
        mx[half * ROWS + r] = __uint_as_float(hit);
        pair_sync(quarter);
        hit |= __float_as_uint(mx[(half ^ 1) * ROWS + r]);
        pair_sync(quarter);
#pragma unroll
        for (int q = 0; q < NP; q++)
          if ((hit >> (2 * q + half)) & 1)
#pragma unroll
            for (int i = 0; i < 32; i++) acc[q][i] = NAN;
      }
#pragma unroll
      for (int j = 0; j < 2; j++) {   // two terms of the products, over the logits: 16 keys are eight columns
        if (more) {
          // Units in which the largest product with a V power is at most 2^14. (A factor: in exp2's argument the power would
          // leave the weight's last bits no room.)
          const float2 unit = make_float2(pow2f(30 - (int)e_run), pow2f(30 - (int)e_run));
          const float4* vexp = reinterpret_cast<const float4*>(smem + G::OFF_VEXP + (slot * SK + half * 32 + j * 16) * 4);
          uint32_t h[8], l[8];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float4 v = vexp[i];
            const float* x = s + 16 * j + 4 * i;
            const float2 w0 = mul2(make_float2(x[0], x[1]), mul2(make_float2(v.x, v.y), unit)), w1 = mul2(make_float2(x[2], x[3]), mul2(make_float2(v.z, v.w), unit));
            split2_scaled(w0.x, w0.y, &h[2 * i], &l[2 * i]);
            split2_scaled(w1.x, w1.y, &h[2 * i + 1], &l[2 * i + 1]);
          }
          tmem_st8(at + 8 * j, h);
          tmem_st8(at + 16 + 8 * j, l);
          if (j == 1) {
            tmem_st_wait();
            tc_fence_before();
            arrive(p_ready + 8 * (it & 1));
          }
        }
      }
      if (NP > 2 && prev) {
        drain(it - 1, 2, acc[2 % NP]);
        drain(it - 1, 3, acc[3 % NP]);
      }
      a_of = a_next;
    }

    // ---- the rows' sums, through shared memory: a row is written whole, and a cluster's CTAs add up theirs, each for its share
    // of the rows
    report_wait();
    pair_sync(quarter);
    ex[half * ROWS + r] = l_run;
    pair_sync(quarter);
    l_run += ex[(half ^ 1) * ROWS + r];
    const bool report = !flags[0] && !flags[1];
    const float back = pow2f((int)e_run - 36);
    float* res = reinterpret_cast<float*>(smem + G::OFF_K);   // (the last product has been read, so the panels are free)
    float* stats = reinterpret_cast<float*>(smem + G::OFF_STATS);
    float* weight = reinterpret_cast<float*>(smem + G::OFF_KRAW);   // [8][ROWS]: what a CTA's sums count in a row
    softmax_sync();
    if (half == 0) stats[r] = m_run, stats[ROWS + r] = l_run;
#pragma unroll
    for (int q = 0; q < NP; q++)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const uint32_t chunk = q * 16 + half * 8 + i;
        *reinterpret_cast<float4*>(res + r * D + ((chunk ^ (r & 7)) << 2)) = make_float4(acc[q][4 * i] * back, acc[q][4 * i + 1] * back, acc[q][4 * i + 2] * back, acc[q][4 * i + 3] * back);
      }
    if (rg.cluster == 1) softmax_sync();
    else cluster_sync();
    const uint32_t share = ROWS / rg.cluster, res_addr = sbase + G::OFF_K, stats_addr = sbase + G::OFF_STATS;
    for (uint32_t i = tid; i < share; i += CW * 32) {
      const uint32_t rr = rank * share + i;
      float m[8], w[8], M = -INFINITY, lsum = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        m[k] = -INFINITY, w[k] = 0.0f;
        if (k < (int)rg.cluster) {
          const uint32_t a = cluster_addr(stats_addr, k);
          m[k] = ld_cluster_f(a + 4 * rr), w[k] = ld_cluster_f(a + 4 * (ROWS + rr));
        }
        M = fmaxf(M, m[k]);
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
        m[k] = m[k] == -INFINITY ? 0.0f : ex2(m[k] - M);
        lsum += w[k] * m[k];
      }
      const bool good = lsum > 0.0f && isfinite(lsum);
      const float inv = good ? __frcp_rn(lsum) : 0.0f;
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (k < (int)rg.cluster) weight[k * ROWS + i] = good ? m[k] * inv : 0.0f;
      uint32_t l;
      if (!good && report && row_of(rr, &l) != NO_ROW) {
        const KeyRange kr = key_range(p, b, l);
        if (kr.hi > kr.lo) atomicCAS(p.fault, FAULT_NONE, FAULT_NONFINITE);
      }
    }
    softmax_sync();
    constexpr int LPR = D < 128 ? D / 4 : 32, VPL = D / 4 / LPR, RPI = CW * 32 / LPR, BATCH = 8 / VPL;   // lanes of a row, rows at once
    const uint32_t d4 = lane % LPR;
    for (uint32_t i0 = warp * (32 / LPR) + lane / LPR; i0 < share; i0 += BATCH * RPI) {
      float4 o[BATCH][VPL];
#pragma unroll
      for (int j = 0; j < BATCH; j++)
#pragma unroll
        for (int c = 0; c < VPL; c++) o[j][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
      for (uint32_t k = 0; k < rg.cluster; k++) {
        const uint32_t from = cluster_addr(res_addr, k);
        float4 v[BATCH][VPL];
#pragma unroll
        for (int j = 0; j < BATCH; j++)
#pragma unroll
          for (int c = 0; c < VPL; c++) {
            const uint32_t rr = rank * share + min(i0 + j * RPI, share - 1);
            v[j][c] = ld_cluster_f4(from + rr * (D * 4) + (((d4 + 32 * c) ^ (rr & 7)) << 4));
          }
#pragma unroll
        for (int j = 0; j < BATCH; j++) {
          const float f = weight[k * ROWS + min(i0 + j * RPI, share - 1)];
#pragma unroll
          for (int c = 0; c < VPL; c++)   // (sums without weight may be anything)
            if (f != 0.0f) o[j][c].x += v[j][c].x * f, o[j][c].y += v[j][c].y * f, o[j][c].z += v[j][c].z * f, o[j][c].w += v[j][c].w * f;
        }
      }
#pragma unroll
      for (int j = 0; j < BATCH; j++) {
        const uint32_t i = i0 + j * RPI, row = i < share ? rows[rank * share + i] : NO_ROW;
        if (row != NO_ROW)
#pragma unroll
          for (int c = 0; c < VPL; c++) *reinterpret_cast<float4*>(p.out + (uint64_t)row * D + 4 * (d4 + 32 * c)) = o[j][c];
      }
    }
    __syncwarp();
    if (rg.cluster > 1) cluster_sync();   // no CTA leaves before the others have read its sums
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(other_regs(D)));
    if (warp == MMA_WARP) {
      // ================ the products ================
      wait(q_ready, 0);
      const uint32_t t0 = __reduce_max_sync(FULL, tmem), rounds = __reduce_max_sync(FULL, stages);   // (uniform registers)
      const uint64_t kh = smem_desc_sw128(sbase + G::OFF_K), kl = kh + NP * (PANEL >> 4);
      const uint64_t vh = smem_desc_sw128(sbase + G::OFF_V), vl = vh + NP * (PANEL >> 4);
      auto logits = [&](uint32_t it) {
        wait(k_ready, it);
        tc_fence_after();
        {
          const uint32_t d = t0 + G::T_S + (it & 1) * 64, qh = t0 + G::T_Q, ql = qh + D / 2;
#pragma unroll 1
          for (int j = 0; j < 3; j++) {   // lo.hi, hi.lo, hi.hi
            const uint32_t a = j == 0 ? ql : qh;
            const uint64_t bd = j == 1 ? kl : kh;
#pragma unroll 1
            for (int q = 0; q < NP; q++) umma_f16_ts4<0, 2>(d, a + 32 * q, bd + q * (PANEL >> 4), IDESC_QK, j | q);
          }
          umma_commit_elected(s_full + 8 * (it & 1));
          umma_commit_elected(k_free);
        }
      };
      if (rounds > 0) logits(0);
      for (uint32_t it = 0; it < rounds; it++) {
        if (it + 1 < rounds) logits(it + 1);
        wait(p_ready + 8 * (it & 1), it >> 1);   // P and V
#pragma unroll 1
        for (int q = 0; q < NP; q++) {
          const uint32_t n = it * NP + q;
          if (n >= 2) wait(o_free + 8 * (n & 1), (n >> 1) - 1);
          tc_fence_after();
          {
            const uint32_t d = t0 + G::T_O + (n & 1) * 64, ph = t0 + G::T_S + (it & 1) * 64;
            // 16 keys: eight columns of P, two groups of eight rows of V. P's second term is times 2^11.
            static_assert(LO_SCALE == 2048.0f, "2^11");
            umma_f16_ts4<16, (2048 >> 4)>(d, ph + 16, vh + q * (PANEL >> 4), IDESC_PV, 0);
            umma_f16_ts4<16, (2048 >> 4), 11>(d, ph, vl + q * (PANEL >> 4), IDESC_PV, 1);
            umma_f16_ts4<16, (2048 >> 4)>(d, ph, vh + q * (PANEL >> 4), IDESC_PV, 1);
            umma_commit_elected(o_full + 8 * (n & 1));
            if (q == NP - 1) umma_commit_elected(v_free);
          }
        }
      }
      report_wait();
      umma_commit_elected(done);
      ptx::mbar_wait_bounded(done, 0, p.wait_limit);
      __syncwarp();
    } else if (warp == LOAD_WARP) {
      // ================ raw stages ================
      if (lane == 0) {
        const uint64_t row0 = p.page_table ? 0 : (uint64_t)b * p.T;
        uint32_t seg = my_first / ts.per_seg, in_seg = my_first - seg * ts.per_seg;
        int32_t page = 0;
        auto lookup = [&](uint32_t s, uint32_t tile) {   // the page of the next tile, read a tile ahead
          page = p.page_table && tile < tiles ? __ldg(p.page_table + (uint64_t)b * p.pages_per_request + s) : 0;
        };
        lookup(seg, 0);
        // A slot is armed again only when it has been read AND its own bytes have come: warps that gave up waiting for them
        // arrive all the same, and a second arrival in a phase that still waits for bytes is an error of the barrier.
        auto reusable = [&](uint32_t full, uint32_t empty, uint32_t use) {
          return use == 0 || (ptx::mbar_wait_bounded(empty, (use - 1) & 1, p.wait_limit) && ptx::mbar_wait_bounded(full, (use - 1) & 1, p.wait_limit));
        };
        bool gone = false;
        uint32_t k_issued = 0, v_issued = 0;
        for (uint32_t it = 0; it < stages && !gone; it++) {
          uint32_t count[SUBS], key[SUBS], bytes_k = 0, bytes_v = 0;
          uint64_t row[SUBS];
#pragma unroll
          for (int s = 0; s < SUBS; s++) {
            const uint32_t tile = it * SUBS + s;
            count[s] = tile < tiles ? tile_rows(ts, in_seg) : 0;
            row[s] = row0 + in_seg * TK;
            key[s] = seg * ts.seg_len + in_seg * TK;
            if (p.page_table) {
              if (count[s] && (page < 0 || (uint32_t)page >= p.pool_pages)) {
                atomicExch(p.fault, FAULT_INVALID_ARGUMENT);   // a page outside the pool: its keys are left out
                count[s] = 0;
              }
              row[s] += (uint64_t)(count[s] ? page : 0) * p.page_tokens;
            }
            if (++in_seg >= ts.per_seg) in_seg = 0, seg++, lookup(seg, tile + 1);
            if (count[s]) bytes_k += TK * KF::PITCH, bytes_v += TK * VF::PITCH;
          }
          const uint32_t ks = it % KRAWS, vs = it % VRAWS, kbar = kraw_full + 8 * ks, vbar = vraw_full + 8 * vs;
          gone = !reusable(kbar, kraw_empty + 8 * ks, it / KRAWS);
          if (gone) break;
          ptx::mbar_arrive_expect_tx(kbar, bytes_k);
          const bool drop = p.drop_first && it == 0;
          if (!drop)
#pragma unroll
            for (int s = 0; s < SUBS; s++)
              if (count[s]) ptx::tma_load_2d(sbase + G::OFF_KRAW + ks * G::KRAW + s * (TK * KF::PITCH), &tmap_k, (int)((hkv * KF::BYTES) / 16 * 2), (int)row[s], kbar);
          gone = !reusable(vbar, vraw_empty + 8 * vs, it / VRAWS);
          k_issued = it + 1;
          if (gone) break;
#pragma unroll
          for (int s = 0; s < SUBS; s++) valid[(it % SLOTS) * SUBS + s] = make_uint2((1u << count[s]) - 1, key[s]);
          ptx::mbar_arrive_expect_tx(vbar, bytes_v);
          v_issued = it + 1;
          if (!drop)
#pragma unroll
            for (int s = 0; s < SUBS; s++)
              if (count[s]) ptx::tma_load_2d(sbase + G::OFF_VRAW + vs * G::VRAW + s * (TK * VF::PITCH), &tmap_v, (int)((hkv * VF::BYTES) / 16 * 2), (int)row[s], vbar);
        }
        if (gone) atomicExch(p.fault, FAULT_WAIT_EXPIRED), flags[1] = 1;
        // No copy is in flight when the block ends.
        for (uint32_t it = k_issued > KRAWS ? k_issued - KRAWS : 0; it < k_issued; it++) ptx::mbar_wait_bounded(kraw_full + 8 * (it % KRAWS), (it / KRAWS) & 1, p.wait_limit);
        for (uint32_t it = v_issued > VRAWS ? v_issued - VRAWS : 0; it < v_issued; it++) ptx::mbar_wait_bounded(vraw_full + 8 * (it % VRAWS), (it / VRAWS) & 1, p.wait_limit);
      }
      __syncwarp();
    } else {
      // ================ raw blocks to operands ================
      const uint32_t uw = warp - FIRST_UNPACK;
      const uint32_t kshift = (hkv * KF::BYTES) & 15, vshift = (hkv * VF::BYTES) & 15;
      using UK = Unpack<D, KQ8>;
      using UV = Unpack<D, VQ8>;
      constexpr int KPW = UK::KPW, GROUPS = UK::GROUPS;
      const uint32_t in_group = lane % KPW, panel = lane / KPW;
      // Is the key there, and does a row of the block see it?
      auto seen = [&](uint32_t it, uint32_t key) {
        const uint2 v = valid[(it % SLOTS) * SUBS + key / TK];
        const uint32_t at = v.y + key % TK;
        return ((v.x >> (key % TK)) & 1) && at >= u_lo && at < u_hi;
      };
      auto key_scales = [&](uint32_t it) {
        wait(kraw_full + 8 * (it % KRAWS), it / KRAWS);
        if (!dead)
#pragma unroll 1
          for (uint32_t u = uw; u < GROUPS; u += UW) {
            const uint32_t key = u * KPW + in_group;
            uint32_t sc[2];
            const uint32_t e = UK::scales(smem + G::OFF_KRAW + (it % KRAWS) * G::KRAW + kshift + panel * 2 * KF::BB + key * KF::PITCH, sc);
            *reinterpret_cast<uint32_t*>(smem + G::OFF_KSC + ((it & 1) * SK * NP + key * NP + panel) * 4) = UK::normed(sc, e);
            if (panel == 0) *reinterpret_cast<float*>(smem + G::OFF_KEXP + ((it % SLOTS) * SK + key) * 4) = pow2f((int)e - 22);
          }
      };
      auto value_scales = [&](uint32_t it) {
        wait(vraw_full + 8 * (it % VRAWS), it / VRAWS);
        if (!dead) {
          uint32_t top = 0, any = 0;
#pragma unroll 1
          for (uint32_t u = uw; u < GROUPS; u += UW) {
            const uint32_t key = u * KPW + in_group;
            uint32_t sc[2], odd = 0;
            const uint32_t e = UV::scales(smem + G::OFF_VRAW + (it % VRAWS) * G::VRAW + vshift + panel * 2 * VF::BB + key * VF::PITCH, sc);
            const bool on = seen(it, key);
#pragma unroll
            for (int i = 0; i < 2; i++) {
              if (on && (sc[i] & 0x7C00u) == 0x7C00u) odd |= (1u << i) << (2 * panel);
              if (!on || (sc[i] & 0x7C00u) == 0x7C00u) sc[i] = 0;
            }
#pragma unroll
            for (int x = KPW; x < 32; x *= 2) odd |= __shfl_xor_sync(FULL, odd, x);
            *reinterpret_cast<uint32_t*>(smem + G::OFF_VSC + ((it % 3) * SK * NP + key * NP + panel) * 4) = UV::normed(sc, e);
            if (panel == 0) {
              *reinterpret_cast<float*>(smem + G::OFF_VEXP + ((it % SLOTS) * SK + key) * 4) = pow2f((int)e - 16);
              smem[G::OFF_ODD + (it % SLOTS) * SK + key] = (uint8_t)odd;
            }
            top = max(top, on ? e : 0u);
            any |= odd;
          }
          top = __reduce_max_sync(FULL, top) | (__any_sync(FULL, any != 0) ? 256u : 0u);
          if (lane == 0) *reinterpret_cast<uint32_t*>(smem + G::OFF_VMAX + ((it % SLOTS) * 8 + uw) * 4) = top;
        }
        arrive(scaled + 8 * (it % SLOTS));
      };
      for (uint32_t it = 0; it <= stages; it++) {
#pragma unroll 1
        for (uint32_t v = 0; v < 2; v++) {   // K of this stage, V of the one before
          const uint32_t st = it - v;
          if (v == 0) {
            if (it < stages) key_scales(it);
            unpack_sync();   // (every warp comes here, also one that has given up)
            if (it == stages) continue;
            if (it == 0) wait(q_ready, 0);   // (q passed through the panels)
          } else {
            if (it < stages) value_scales(it);
            if (it == 0) break;
          }
          if (st > 0) wait(v ? v_free : k_free, st - 1);
          if (!dead) {
            const uint8_t* raw = smem + (v ? G::OFF_VRAW + (st % VRAWS) * G::VRAW + vshift + panel * 2 * VF::BB
                                           : G::OFF_KRAW + (st % KRAWS) * G::KRAW + kshift + panel * 2 * KF::BB);
            const uint32_t* sc = reinterpret_cast<const uint32_t*>(smem + (v ? G::OFF_VSC : G::OFF_KSC)) + (v ? st % 3 : st & 1) * SK * NP + panel;
            uint8_t* hi = smem + (v ? G::OFF_V : G::OFF_K) + panel * PANEL;
            const uint32_t pitch = v ? VF::PITCH : KF::PITCH;
#pragma unroll 1
            for (uint32_t u = uw; u < 2 * GROUPS; u += UW) {
              const uint32_t key = (u >> 1) * KPW + in_group;
              if (KQ8 == VQ8 || v == 0) UK::block(raw + key * pitch, u & 1, sc[key * NP], hi, hi + NP * PANEL, key);
              else UV::block(raw + key * pitch, u & 1, sc[key * NP], hi, hi + NP * PANEL, key);
            }
            ptx::fence_proxy_async();
          }
          arrive(v ? p_ready + 8 * (st & 1) : k_ready);
          arrive(v ? vraw_empty + 8 * (st % VRAWS) : kraw_empty + 8 * (st % KRAWS));
        }
      }
      report_wait();
    }
    if (rg.cluster > 1) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  }
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

template <int D, bool KQ8, bool VQ8, bool CAP>
int32_t launch_rows(AionCudaDevice* dev, const AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, uint64_t max_keys) {
  using G = RowsGeom<D, KQ8, VQ8>;
  auto kernel = attn_qcache_rows_kernel<D, KQ8, VQ8, CAP>;
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
  // cost a third of a stage for each of them.
  rg.cluster = 1;
  double best = 1e30;
  for (uint32_t c = 1, i = 0; c <= 8 && max_keys >= (uint64_t)c * (c > 1 ? 4 : 0) * SK; c *= 2, i++) {
    const double cost = std::ceil((double)units / held[i]) * (std::ceil((double)max_keys / (c * SK)) + 4.0 + (c > 1 ? 0.35 * c : 0.0));
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
  dev->debug_qcache = {AION_CUDA_QCACHE_KERNEL_ROWS, rg.cluster, 0u};
  return AION_CUDA_OK;
}

}  // namespace

int32_t attention_qcache_rows(AionCudaDevice* dev, const AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, uint64_t max_keys) {
  const bool kq8 = p.k_dtype == AION_CUDA_DTYPE_Q8_0, vq8 = p.v_dtype == AION_CUDA_DTYPE_Q8_0;
  // (A soft cap in a kernel of its own: its instructions in the loop cost the others 11 %.)
#define AION_QROWS_AS(D, K, V) return p.soft_cap > 0.0f ? launch_rows<D, K, V, true>(dev, p, tk, tv, max_keys) : launch_rows<D, K, V, false>(dev, p, tk, tv, max_keys);
#define AION_QROWS(D)                                          \
  if (kq8 && vq8) AION_QROWS_AS(D, true, true)                 \
  if (kq8) AION_QROWS_AS(D, true, false)                       \
  if (vq8) AION_QROWS_AS(D, false, true)                       \
  AION_QROWS_AS(D, false, false)
  switch (p.Dk) {
    case 64: AION_QROWS(64)
    case 128: AION_QROWS(128)
    default: AION_QROWS(256)
  }
#undef AION_QROWS
#undef AION_QROWS_AS
}

}  // namespace aion
