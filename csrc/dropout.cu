// Dropout with a counter-based generator, and with the sum of the residual stream where there is one.
//
//   y[i] = residual[i] + (keep(i) ? x[i] / (1 - p) : 0),   keep(i): the i % 8-th 16 bits of Philox4x32-10 at i / 8 are p 2^16 or more.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) makes 128 bits of a key and a 128-bit
// counter by ten rounds of two multiplications.  The key is the seed, the counter the element's number / 8, the step and the place
// in the model, so a mask is made again wherever it is needed (the backward pass, a recomputed layer) and never stored.  A thread makes
// the bits of one 16-byte vector: sixteen bits an element are one generator call per vector, about 40 instructions for what is
// loaded and stored with two; 32 would be twice that, more than memory leaves time for.  The round keys are the same in every thread.
// The gradient is the same operator on dy.

#include <initializer_list>

#include "common.cuh"
#include "tpb.h"

namespace tpb {

int sm_count();

struct Dropout {
  const __nv_bfloat16 *x, *residual;
  __nv_bfloat16* y;
  const long long* seed;                     // {key, step}
  unsigned long long n;
  unsigned threshold, site;                  // the threshold in steps of 2^-16, up to 2^16
  float up;
};

struct PhiloxKeys {
  uint32_t a[10], b[10];
  __device__ __forceinline__ explicit PhiloxKeys(unsigned long long key) {
    a[0] = (uint32_t)key;
    b[0] = (uint32_t)(key >> 32);
#pragma unroll
    for (int i = 1; i < 10; ++i) {
      a[i] = a[i - 1] + 0x9E3779B9u;
      b[i] = b[i - 1] + 0xBB67AE85u;
    }
  }
};
__device__ __forceinline__ uint4 philox(uint4 c, const PhiloxKeys& k) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const unsigned long long p = (unsigned long long)c.x * 0xD2511F53u, q = (unsigned long long)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(q >> 32) ^ c.y ^ k.a[i], (uint32_t)q, (uint32_t)(p >> 32) ^ c.w ^ k.b[i], (uint32_t)p);
  }
  return c;
}

// The two elements of a word, the low half first: compared with the threshold in the upper half of a word (65536: nothing stays).
__device__ __forceinline__ uint32_t drop_pair(uint32_t x, uint32_t bits, unsigned long long least, float up, const uint32_t* residual) {
  const float2 v = unpack_bf16(x);
  float a = (bits << 16) >= least ? mul_exact(v.x, up) : 0.f;
  float b = bits >= least ? mul_exact(v.y, up) : 0.f;
  if (residual) {
    const float2 r = unpack_bf16(*residual);
    a = add_exact(a, r.x);
    b = add_exact(b, r.y);
  }
  return pack_bf16(a, b);
}

constexpr int DROP_AHEAD = 4;

template <bool RES>
__global__ void __launch_bounds__(256)
dropout_kernel(const Dropout p) {
  if (!chain_begin()) return;
  const PhiloxKeys keys(p.seed[0]);
  const uint32_t step = (uint32_t)p.seed[1];
  const unsigned long long vecs = p.n / 8, stride = (unsigned long long)gridDim.x * 256, least = (unsigned long long)p.threshold << 16;
  const uint4 *x = reinterpret_cast<const uint4*>(p.x), *res = reinterpret_cast<const uint4*>(p.residual);
  uint4* y = reinterpret_cast<uint4*>(p.y);
  for (unsigned long long i0 = blockIdx.x * 256ull + threadIdx.x; i0 < vecs; i0 += DROP_AHEAD * stride) {
    uint4 v[DROP_AHEAD], r[DROP_AHEAD];
#pragma unroll
    for (int j = 0; j < DROP_AHEAD; ++j) {
      const unsigned long long i = i0 + j * stride;
      if (i < vecs) {
        v[j] = x[i];
        if (RES) r[j] = res[i];
      }
    }
#pragma unroll
    for (int j = 0; j < DROP_AHEAD; ++j) {
      const unsigned long long i = i0 + j * stride;
      if (i >= vecs) break;
      const uint4 bits = philox(make_uint4((uint32_t)i, (uint32_t)(i >> 32), step, p.site), keys);
      y[i] = make_uint4(drop_pair(v[j].x, bits.x, least, p.up, RES ? &r[j].x : nullptr), drop_pair(v[j].y, bits.y, least, p.up, RES ? &r[j].y : nullptr),
                        drop_pair(v[j].z, bits.z, least, p.up, RES ? &r[j].z : nullptr), drop_pair(v[j].w, bits.w, least, p.up, RES ? &r[j].w : nullptr));
    }
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x < p.n % 8) {      // what does not fill a vector
    const unsigned long long i = vecs * 8 + threadIdx.x;
    const uint4 bits = philox(make_uint4((uint32_t)vecs, (uint32_t)(vecs >> 32), step, p.site), keys);
    const int e = threadIdx.x;
    const uint32_t w = e < 2 ? bits.x : e < 4 ? bits.y : e < 6 ? bits.z : bits.w;
    float a = (e & 1 ? w : w << 16) >= least ? mul_exact(__bfloat162float(p.x[i]), p.up) : 0.f;
    if (RES) a = add_exact(a, __bfloat162float(p.residual[i]));
    p.y[i] = __float2bfloat16(a);
  }
}

}  // namespace tpb

using namespace tpb;

// y = (residual +) dropout of n bf16 numbers (16-byte aligned; residual null: none).  seed {key, step} int64 in device memory;
// threshold: p in steps of 2^-16, site: the place in the model.
extern "C" int tpb_dropout(const void* x, const void* residual, void* y, const long long* seed, long long n, int threshold, unsigned site,
                           void* stream) {
  if (n < 0 || threshold < 0 || threshold > 65536) return -2;
  for (const void* a : {x, residual, (const void*)y})
    if (reinterpret_cast<uintptr_t>(a) % 16) return -2;
  if (n == 0) return 0;
  Dropout p = {static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(residual), static_cast<__nv_bfloat16*>(y), seed,
               (unsigned long long)n, (unsigned)threshold, site, threshold < 65536 ? 65536.f / (65536 - threshold) : 0.f};
  const long long blocks = (n / 8 + 255) / 256, most = 8LL * sm_count();
  const int grid = (int)(blocks < 1 ? 1 : blocks < most ? blocks : most);
  if (residual) chain(dropout_kernel<true>, grid, 256, 0, static_cast<cudaStream_t>(stream), p);
  else chain(dropout_kernel<false>, grid, 256, 0, static_cast<cudaStream_t>(stream), p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
