// What the two tensor-core kernels over a quantized cache share: how a head row lies in shared memory, how a context is
// cut into tiles, and the arithmetic on fragments.
#pragma once

#include "attention_device.cuh"
#include "cache_geom.cuh"

namespace aion {
namespace qcache {

constexpr uint32_t FULL = 0xFFFFFFFFu;
constexpr int TK = TILE_KEYS;       // keys of a tile

template <int D, bool Q8>
struct RowFmt {
  static constexpr int BB = Q8 ? Q8_BYTES : Q4_BYTES;
  static constexpr int BYTES = D / QK * BB;          // one head row
  static constexpr int CHUNKS = Q8 ? 17 : 9;         // copies of CHUNK bytes
  static constexpr int CHUNK = D / 16;
  static constexpr int PITCH = Q8 ? (D == 64 ? 80 : D == 128 ? 144 : 272) : (D == 64 ? 48 : D == 128 ? 80 : 144);
  static_assert(CHUNKS * CHUNK == BYTES && PITCH % CHUNK == 0 && PITCH >= BYTES && (PITCH / 4) % 8 == 4, "row layout");
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t a, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }

__device__ __forceinline__ CacheGeom geom_of(const AttnParams& p) {
  return CacheGeom{p.page_table, p.T, p.page_tokens, p.pages_per_request, p.pool_pages, p.rolling};
}
__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// D = A . B + C with a C of its own.
__device__ __forceinline__ void mma_f16_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                             float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ float ex2(float x) {   // 2^x to 2 units in the last place; 0 for -infinity
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float half_bits(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }
__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Two terms of f16 for a pair of f32 values: x = hi + lo to 22 bits. The remainder is taken by an operation that
// reads the f16 term as it is (times -1) (on the FMA pipe; a conversion back to f32 would go to the busier ALU pipe).
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  const uint32_t h = pack_half2(a, b);
  float la, lb;   // x - hi
  asm("{.reg .b16 l, h, m;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 m, 0xBC00;\n\tfma.rn.f32.f16 %0, l, m, %3;\n\tfma.rn.f32.f16 %1, h, m, %4;\n\t}"
      : "=f"(la), "=f"(lb)
      : "r"(h), "f"(a), "f"(b));
  *hi = h;
  *lo = pack_half2(la, lb);
}
// The same with the second term times 2^11, for weights: they reach down to where f16 has no more bits (a small weight, or small
// values beside large ones), and so scaled the second term keeps eleven bits where the first one has none left. Together they are
// good to 2^-23 of x down to 2^-14, and to 2^-37 below that. Its products have a sum of their own.
constexpr float LO_SCALE = 2048.0f;
__device__ __forceinline__ void split2_scaled(float a, float b, uint32_t* hi, uint32_t* lo) {
  const uint32_t h = pack_half2(a, b);
  float la, lb;   // 2^11 x - 2^11 hi
  asm("{.reg .b16 l, h, m;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 m, 0xE800;\n\tfma.rn.f32.f16 %0, l, m, %3;\n\tfma.rn.f32.f16 %1, h, m, %4;\n\t}"
      : "=f"(la), "=f"(lb)
      : "r"(h), "f"(a * LO_SCALE), "f"(b * LO_SCALE));
  *hi = h;
  *lo = pack_half2(la, lb);
}

// cap * tanh(x / cap) of N logits. Up to |x| = cap, where capped logits mostly lie, tanh is the sixth convergent of
// Lambert's continued fraction z / (1 + z^2 / (3 + z^2 / (5 + ...))), whose error at z = 1 is 7e-10; beyond it tanhf.
// (Five rows over a ring of 1023 keys: 18 us, with tanhf throughout 25.)
// (1 / cap of a cap below f32's normal range is held at f32's largest number: a logit of zero stays one.)
__device__ __forceinline__ float inverse_cap(float cap) { return fminf(1.0f / cap, FLT_MAX); }
template <int N>
__device__ __forceinline__ void cap_logits(float (&x)[N], float cap, float inv_cap) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i++) top = fmaxf(top, fabsf(x[i]));
  if (__any_sync(FULL, top > cap)) {
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = cap * tanhf(x[i] * inv_cap);
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float z = x[i] * inv_cap, w = z * z;
      const float num = fmaf(w, fmaf(w, 21.0f, 1260.0f), 10395.0f), den = fmaf(w, fmaf(w, w + 210.0f, 4725.0f), 10395.0f);
      x[i] = x[i] * __fdividef(num, den);
    }
  }
}

// Two f32 products or sums in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)));
  return *reinterpret_cast<const float2*>(&d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<const uint64_t*>(&a)), "l"(*reinterpret_cast<const uint64_t*>(&b)), "l"(*reinterpret_cast<const uint64_t*>(&c)));
  return *reinterpret_cast<const float2*>(&d);
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  const float2 u = make_float2(x, y), v = make_float2(a, b);
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<const uint64_t*>(&u)), "l"(*reinterpret_cast<const uint64_t*>(&v)));
  const float2 r = *reinterpret_cast<const float2*>(&d);
  x = r.x, y = r.y;
}

// Which dimension of a block the lane index u (t of a key row's words) reaches with code i of its word(s).
// K words: q4_0 one word of eight nibbles per lane t; q8_0 two words, u = t and t + 4, of four bytes.
__host__ __device__ constexpr int pair_byte(bool q8, bool second, int u, int j) {
  // byte j of word u of the block's codes; in a pair's first block word 0 is put together from the codes' first
  // and last two bytes (they share words with the two scales)
  const int n = q8 ? 32 : 16;
  return second ? 4 * u + j : u ? 4 * u - 2 + j : j < 2 ? j : n - 4 + j;
}

// 0x6400 | n is 1024 + n, 0x6400 | 16 n is 1024 + 16 n: both leave n - 8 exactly.
__device__ __forceinline__ void unpack_q4(uint32_t w, uint32_t (&x)[4]) {
  x[0] = h2_add((w & 0x000F000Fu) | 0x64006400u, 0xE408E408u);
  x[1] = h2_fma((w & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u);
  w >>= 8;
  x[2] = h2_add((w & 0x000F000Fu) | 0x64006400u, 0xE408E408u);
  x[3] = h2_fma((w & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u);
}
__device__ __forceinline__ void unpack_q8(uint32_t w, uint32_t* r0, uint32_t* r1) {
  w ^= 0x80808080u;
  // 0x6400 | u is 1024 + u: minus 1152 leaves the signed code, exactly
  *r0 = h2_add(__byte_perm(w, 0x64646464u, 0x4140), 0xE480E480u);
  *r1 = h2_add(__byte_perm(w, 0x64646464u, 0x4342), 0xE480E480u);
}

}  // namespace qcache

// Many query rows (attention_qcache_rows.cu): K and V by boxes of 16 rows of the head's bytes.
int32_t attention_qcache_rows(AionCudaDevice* dev, const AttnParams& p, const CUtensorMap& tk, const CUtensorMap& tv, uint64_t max_keys);
}  // namespace aion
