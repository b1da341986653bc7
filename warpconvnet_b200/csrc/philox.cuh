// The random bits of dropout: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011), a
// bijection of a 128-bit counter under a 64-bit key, so that an element's bits follow from the seed and the element's place alone:
// the gradient makes the same ones again and no mask is kept.  The key is the seed; the counter (column / 8, row, row >> 32, 0)
// gives 16 bits to each of eight columns of a row, low halves of words first.  Sixteen bits an element because 32 would be twice the rounds,
// which take as long as HBM then (115 million elements in 16 bits: some 30 us at eight elements a call, the rows themselves
// 70); a probability is therefore a multiple of 2^-16, and the factor of what is kept goes by that multiple.
#pragma once
#include "wcn_common.cuh"

// What is dropped: elements whose 16 bits are below `least`.
struct wcn_drop {
  uint32_t least;         // 0: nothing
  float scale;            // 65536 / (65536 - least); 0 where everything is dropped
  uint64_t seed;
  const int64_t* at;      // where the seed is (null: `seed`)
};

static inline wcn_drop wcn_make_drop(uint32_t least, int64_t seed, const int64_t* at) {
  return {least, least < 65536u ? 65536.f / (float)(65536u - least) : 0.f, (uint64_t)seed, at};
}

#ifdef __CUDACC__
namespace {

__device__ __forceinline__ uint64_t drop_seed(const wcn_drop& d) { return d.at ? (uint64_t)__ldg(d.at) : d.seed; }

// The keys of the ten rounds: they follow from the seed alone.  (Where registers are short they are kept in shared memory.)
struct alignas(16) PhiloxKeys {
  uint32_t a[10], b[10];
};
__device__ __forceinline__ PhiloxKeys philox_keys(uint64_t seed) {
  PhiloxKeys k;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    k.a[r] = (uint32_t)seed + r * 0x9E3779B9u;
    k.b[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
  }
  return k;
}
__device__ __forceinline__ uint4 philox_eight(const PhiloxKeys& k, uint32_t block, uint64_t row) {
  uint32_t c0 = block, c1 = (uint32_t)row, c2 = (uint32_t)(row >> 32), c3 = 0;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k.a[r];
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k.b[r];
    c3 = (uint32_t)p0;
  }
  return make_uint4(c0, c1, c2, c3);
}
// Eight numbers of a row, columns 8 * block on: zero (whatever they were) or times the scale.  (The bits are compared where they
// stand in a word's upper half: what is below them there decides nothing against a bound that ends in ones.)  Not for `least` 0.
__device__ __forceinline__ void drop_eight(const wcn_drop& d, const PhiloxKeys& keys, uint32_t block, uint64_t row, float2 (&v)[4]) {
  const uint4 w = philox_eight(keys, block, row);
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  const uint32_t bound = (d.least << 16) - 1u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 y = __fmul2_rn(v[i], make_float2(d.scale, d.scale));
    v[i].x = (words[i] << 16) > bound ? y.x : 0.f;
    v[i].y = words[i] > bound ? y.y : 0.f;
  }
}

}  // namespace
#endif
