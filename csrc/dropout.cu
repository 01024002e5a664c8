// Dropout with a counter-based generator, and with the sum of the residual stream where there is one.
//
//   y[i] = residual[i] + (keep(i) ? x[i] / (1 - p) : 0),   keep(i): the i % 8-th 16 bits of Philox4x32-10 at i / 8 are p 2^16 or more.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) makes 128 bits of a key and a 128-bit
// counter by ten rounds of two multiplications.  The key is the seed, the counter the element's number / 8, the step and the place
// in the model, so a mask is made again wherever it is needed (the backward pass, a recomputed layer) and never stored.  A thread makes
// the bits of one 16-byte vector at a time: sixteen bits an element are one generator call per vector, about 40 instructions for what is
// loaded and stored with two; 32 would be twice that, more than memory leaves time for.  The gradient is the same operator on dy.
// Memory bounds it: 16384 x 4096 numbers 41.8 us, with a residual 60.0 (41.0 and 61.5 at a copy's rate).

#include <initializer_list>

#include "common.cuh"
#include "tpb.h"

namespace tpb {

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

// The two elements of a word, the low half first: they stay where their bits, in the upper half of a word, are above `most`.
__device__ __forceinline__ uint32_t drop_pair(uint32_t x, uint32_t bits, uint32_t most, float up, const uint32_t* residual) {
  const float2 v = unpack_bf16(x);
  float a = (bits << 16) > most ? mul_exact(v.x, up) : 0.f;
  float b = bits > most ? mul_exact(v.y, up) : 0.f;
  if (residual) {
    const float2 r = unpack_bf16(*residual);
    a = add_exact(a, r.x);
    b = add_exact(b, r.y);
  }
  return pack_bf16(a, b);
}

constexpr int DROP_THREADS = 256;
// Vectors to a thread: six of tensors from 2^24 numbers on, so that enough is under way, three of smaller ones, for more threads.  us, 3 / 6: 333 x 2048
// 1.7 / 3.5, 2048 x 4096 with a residual 9.5 / 10.5, 8197 x 5120 30.3 / 27.3, 16384 x 4096 46.6 / 41.8, with a residual 59.6 / 60.0.  (Four in
// registers of a persistent grid 2.2, -, 32.4, 49, 69.)
constexpr int DROP_FEW = 3, DROP_MANY = 6;
constexpr unsigned long long DROP_MANY_FROM = 1ull << 24;

__device__ __forceinline__ void drop_ask(uint4* dst, const uint4* src, bool has) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(has ? 16 : 0) : "memory");
}

// A thread takes VECS vectors, DROP_THREADS apart, and leaves.  It asks for all of them first, into places of its own in shared memory, and
// makes the bits of the first while they come.
template <bool RES, int VECS>
__global__ void __launch_bounds__(DROP_THREADS, VECS > DROP_FEW ? 4 : 5)
dropout_kernel(const Dropout p) {
  __shared__ uint4 mem[VECS * (RES ? 2 : 1)][DROP_THREADS];
  if (!chain_begin()) return;
  const unsigned long long vecs = p.n / 8, i0 = (unsigned long long)blockIdx.x * (VECS * DROP_THREADS) + threadIdx.x;
  const uint4 *x = reinterpret_cast<const uint4*>(p.x), *res = reinterpret_cast<const uint4*>(p.residual);
  uint4* y = reinterpret_cast<uint4*>(p.y);
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    const unsigned long long i = i0 + j * DROP_THREADS;
    drop_ask(&mem[j][threadIdx.x], x + (i < vecs ? i : 0), i < vecs);
    if (RES) drop_ask(&mem[VECS + j][threadIdx.x], res + (i < vecs ? i : 0), i < vecs);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  const PhiloxKeys keys(p.seed[0]);
  const uint32_t step = (uint32_t)p.seed[1], most = (p.threshold << 16) - 1;
#pragma unroll
  for (int j = 0; j < VECS; ++j) {
    const unsigned long long i = i0 + j * DROP_THREADS;
    if (i >= vecs) break;
    const uint4 bits = philox(make_uint4((uint32_t)i, (uint32_t)(i >> 32), step, p.site), keys);
    if (j == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    const uint4 v = mem[j][threadIdx.x], r = RES ? mem[VECS + j][threadIdx.x] : make_uint4(0, 0, 0, 0);
    y[i] = make_uint4(drop_pair(v.x, bits.x, most, p.up, RES ? &r.x : nullptr), drop_pair(v.y, bits.y, most, p.up, RES ? &r.y : nullptr),
                      drop_pair(v.z, bits.z, most, p.up, RES ? &r.z : nullptr), drop_pair(v.w, bits.w, most, p.up, RES ? &r.w : nullptr));
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");      // (of a thread without a vector: zeros on their way to its places)
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x < p.n % 8) {      // what does not fill a vector
    const unsigned long long i = vecs * 8 + threadIdx.x;
    const uint4 bits = philox(make_uint4((uint32_t)vecs, (uint32_t)(vecs >> 32), step, p.site), keys);
    const int e = threadIdx.x;
    const uint32_t w = e < 2 ? bits.x : e < 4 ? bits.y : e < 6 ? bits.z : bits.w;
    float a = (e & 1 ? w : w << 16) > most ? mul_exact(__bfloat162float(p.x[i]), p.up) : 0.f;
    if (RES) a = add_exact(a, __bfloat162float(p.residual[i]));
    p.y[i] = __float2bfloat16(a);
  }
}

template <bool RES, int VECS>
static cudaError_t launch_dropout_by(const Dropout& p, cudaStream_t stream) {
  const unsigned long long per = 8ull * VECS * DROP_THREADS, blocks = (p.n + per - 1) / per;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  return chain(dropout_kernel<RES, VECS>, (unsigned)blocks, DROP_THREADS, 0, stream, p);
}
template <bool RES>
static cudaError_t launch_dropout(const Dropout& p, cudaStream_t stream) {
  return p.n < DROP_MANY_FROM ? launch_dropout_by<RES, DROP_FEW>(p, stream) : launch_dropout_by<RES, DROP_MANY>(p, stream);
}

}  // namespace tpb

using namespace tpb;

// y = (residual +) dropout of n bf16 numbers (16-byte aligned; residual null: none).  seed {key, step} int64 in device memory;
// threshold: p in steps of 2^-16, at least 1; site: the place in the model.
extern "C" int tpb_dropout(const void* x, const void* residual, void* y, const long long* seed, long long n, int threshold, unsigned site,
                           void* stream) {
  if (n < 0 || threshold < 1 || threshold > 65536) return -2;
  for (const void* a : {x, residual, (const void*)y})
    if (reinterpret_cast<uintptr_t>(a) % 16) return -2;
  if (n == 0) return 0;
  Dropout p = {static_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(residual), static_cast<__nv_bfloat16*>(y), seed,
               (unsigned long long)n, (unsigned)threshold, site, threshold < 65536 ? 65536.f / (65536 - threshold) : 0.f};
  const cudaError_t launched = residual ? launch_dropout<true>(p, static_cast<cudaStream_t>(stream))
                                        : launch_dropout<false>(p, static_cast<cudaStream_t>(stream));
  const cudaError_t e = launched != cudaSuccess ? launched : cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
