// Norms of the query and key heads of a fused projection with the position rotation in the same pass, and their gradient.
//
//   y = R(p) (w * x r),  r = (mean(x^2) + eps)^-1/2 over the d columns of a head;  w optional;  R(p) turns pairs of the leading
//   `rot` columns by the angles of position p: columns (i, i + rot / 2), or neighbours (2i, 2i + 1);
//   g = R(p)^T dy,  dw = sum over tokens and heads of g x r,  dx = r w g - x r^3 mean(w g x).
//
// A head is read once and written once, two or three bf16 numbers in and out for each product, so memory bounds both directions.  A lane
// holds two 16-byte vectors of a head, the two that are turned with one another: the rotation needs no neighbour, and the sums of a
// head of 128 columns are three shuffles over eight lanes.  Statistics, products and sums are fp32, two side by side in packed
// instructions; results are rounded once.  The gradient takes r from x again (x has to be read there anyway) and, of the weights, adds
// up in registers over all heads that a thread sees, then over the CTA's warps and over the CTAs, in an order that only the sizes decide.
// What bounds them in practice is how much is under way: both read into shared memory with copies that a thread asks for far ahead and
// waits for by itself (no barriers).  One B200, inputs larger than L2, us and the time at a copy's rate: 8192 tokens of 32 / 8 heads of 128 with
// weights 28.8 (25.6) forward, 53.7 (43.6) backward; 32768 of 64 / 8 179 (184) and 311 (297); 48 tokens 2.3 and 7.9.

#include <atomic>
#include <initializer_list>

#include "common.cuh"
#include "tpb.h"

namespace tpb {

int sm_count();

struct QkNorm {
  const __nv_bfloat16* x;                    // [tokens, (hq + 2 hkv) * d], rows ld apart
  long long ld;
  const __nv_bfloat16 *w[2];                 // of queries, of keys; null: ones
  const float *cos, *sin;                    // [table, rot / 2]
  const int* pos;                            // [tokens]; null: token % seq
  int* status;
  __nv_bfloat16* y[2];                       // forward: [tokens, hq or hkv, d]
  const __nv_bfloat16 *dy[3];                // backward: the same, and of the values
  __nv_bfloat16* dx;                         // [tokens, (hq + 2 hkv) * d]
  float* parts;                              // [CTAs][2][d]
  int tokens, seq, table, d, rot;
  int heads[2];
  float eps;
};

constexpr int QK_THREADS = 256, QK_WARPS = QK_THREADS / 32;

// Where a lane's two vectors lie in a head, and whether they are turned.
struct QkLane {
  int a, b;
  bool has, turned;
  __device__ __forceinline__ QkLane(int j, int d, int rot) {
    has = j < d / 16;
    turned = j < rot / 16;
    const int m = j - rot / 16;
    a = turned ? 8 * j : rot + 8 * m;
    b = turned ? rot / 2 + 8 * j : rot + (d - rot) / 2 + 8 * m;
  }
};

// A lane's sixteen columns as the first and the second numbers of its eight pairs, two of them side by side for packed arithmetic.
struct QkPairs {
  f32x2 u[4], v[4];
};
template <bool PAIRS>
__device__ __forceinline__ QkPairs qk_unpack(const uint4& a, const uint4& b) {
  auto lo = [](uint32_t x, uint32_t y) { return f2_pack_bits(x << 16, y << 16); };
  auto hi = [](uint32_t x, uint32_t y) { return f2_pack_bits(x & 0xffff0000u, y & 0xffff0000u); };
  auto both = [](uint32_t x) { return f2_pack_bits(x << 16, x & 0xffff0000u); };
  QkPairs f;
  if (PAIRS) {
    f.u[0] = lo(a.x, a.y); f.u[1] = lo(a.z, a.w); f.u[2] = lo(b.x, b.y); f.u[3] = lo(b.z, b.w);
    f.v[0] = hi(a.x, a.y); f.v[1] = hi(a.z, a.w); f.v[2] = hi(b.x, b.y); f.v[3] = hi(b.z, b.w);
  } else {
    f.u[0] = both(a.x); f.u[1] = both(a.y); f.u[2] = both(a.z); f.u[3] = both(a.w);
    f.v[0] = both(b.x); f.v[1] = both(b.y); f.v[2] = both(b.z); f.v[3] = both(b.w);
  }
  return f;
}
template <bool PAIRS>
__device__ __forceinline__ void qk_store(const QkPairs& f, __nv_bfloat16* a, __nv_bfloat16* b) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float u0, u1, v0, v1;
    f2_unpack(f.u[i], u0, u1);
    f2_unpack(f.v[i], v0, v1);
    if (PAIRS) {
      w[2 * i] = pack_bf16(u0, v0);
      w[2 * i + 1] = pack_bf16(u1, v1);
    } else {
      w[i] = pack_bf16(u0, u1);
      w[4 + i] = pack_bf16(v0, v1);
    }
  }
  *reinterpret_cast<uint4*>(a) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(b) = make_uint4(w[4], w[5], w[6], w[7]);
}

// cos and sin of a lane's eight pairs.
struct QkAngles {
  f32x2 c[4], s[4];
};
template <bool PAIRS>
__device__ __forceinline__ void qk_angles(const QkNorm& p, const QkLane& l, int t, QkAngles& x) {
  int at = p.pos ? p.pos[t] : t % p.seq;
  if ((unsigned)at >= (unsigned)p.table) {
    report(p.status, kBadArgument, 81);
    at = at < 0 ? 0 : p.table - 1;
  }
  if (!l.turned) return;
  const long long row = (long long)at * (p.rot / 2);
  const int i = PAIRS ? l.a / 2 : l.a, k = PAIRS ? l.b / 2 : l.a + 4;
  const float4 c0 = *reinterpret_cast<const float4*>(p.cos + row + i), c1 = *reinterpret_cast<const float4*>(p.cos + row + k);
  const float4 s0 = *reinterpret_cast<const float4*>(p.sin + row + i), s1 = *reinterpret_cast<const float4*>(p.sin + row + k);
  x.c[0] = f2_pack(c0.x, c0.y); x.c[1] = f2_pack(c0.z, c0.w); x.c[2] = f2_pack(c1.x, c1.y); x.c[3] = f2_pack(c1.z, c1.w);
  x.s[0] = f2_pack(s0.x, s0.y); x.s[1] = f2_pack(s0.z, s0.w); x.s[2] = f2_pack(s1.x, s1.y); x.s[3] = f2_pack(s1.z, s1.w);
}
template <bool BACK>
__device__ __forceinline__ void qk_turn(QkPairs& f, const QkAngles& x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f32x2 u = f.u[i], v = f.v[i];
    f.u[i] = BACK ? f2_fma(v, x.s[i], f2_mul(u, x.c[i])) : f2_sub(f2_mul(u, x.c[i]), f2_mul(v, x.s[i]));
    f.v[i] = BACK ? f2_sub(f2_mul(v, x.c[i]), f2_mul(u, x.s[i])) : f2_fma(u, x.s[i], f2_mul(v, x.c[i]));
  }
}
__device__ __forceinline__ QkPairs qk_times(const QkPairs& f, const QkPairs& g) {
  QkPairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.u[i] = f2_mul(f.u[i], g.u[i]);
    r.v[i] = f2_mul(f.v[i], g.v[i]);
  }
  return r;
}
__device__ __forceinline__ float qk_dot(const QkPairs& f, const QkPairs& g) {
  f32x2 a = f2_mul(f.u[0], g.u[0]), b = f2_mul(f.v[0], g.v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    a = f2_fma(f.u[i], g.u[i], a);
    b = f2_fma(f.v[i], g.v[i], b);
  }
  float lo, hi;
  f2_unpack(f2_add(a, b), lo, hi);
  return lo + hi;
}

template <int GROUP>
__device__ __forceinline__ float qk_sum(float v) {
#pragma unroll
  for (int o = 1; o < GROUP; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sixteen bytes to this thread's own place in shared memory (zeros, if there is nothing to be had): what a thread asks for only it reads,
// so its own wait is all that has to lie between.
__device__ __forceinline__ void qk_ask(uint4* dst, const void* src, bool has) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(has ? 16 : 0) : "memory");
}
__device__ __forceinline__ void qk_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int BUT>
__device__ __forceinline__ void qk_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(BUT) : "memory");
}

constexpr int QF_CTAS = 4;                   // of the forward kernel to an SM (64 registers)
// Of the gradient's: heads of a warp at a time (in steps of 32 / GROUP), CTAs to an SM, stages of a thread's.  8192 tokens of 32 / 8 heads, 32768
// of 64 / 8, us: 2, 2, 2 54 and 311;  2, 2, 3 55 and 313;  3, 2, 2 56 and 318;  4, 1, 3 66 and 358;  1, 2, 6 70 and 382 (with the values behind).  There a unit is
// exactly the eight keys of a token; where it is not, most of it is empty: 8192 tokens of 7 / 1 heads 24.4 (8.3 at a copy's rate), of 10 / 2 of 256 40.1 (25.6).
constexpr int QB_STEPS = 2, QB_CTAS = 2, QB_STAGES = 2;

// A warp takes up to STEPS x 32 / GROUP heads of a token, queries and keys, and leaves.  What it reads is all asked for first, into shared
// memory: in registers (four vectors to a thread) too little is under way (8192 tokens of 32 / 8 heads 33.2 us, 32768 of 64 / 8 213).
template <int GROUP, bool PAIRS, int STEPS>
__global__ void __launch_bounds__(QK_THREADS, QF_CTAS)
qk_norm_fwd_kernel(const QkNorm p, unsigned units, unsigned blocks, int steps) {
  constexpr int HPW = 32 / GROUP;
  __shared__ uint4 mem[STEPS * 2][QK_THREADS];
  if (!chain_begin()) return;
  const unsigned unit = blockIdx.x * QK_WARPS + warp_index();
  if (unit >= units) return;
  const int lane = threadIdx.x & 31, t = unit / blocks, h0 = (unit - t * blocks) * steps * HPW + lane / GROUP;
  const int all = p.heads[0] + p.heads[1];
  const QkLane l(lane % GROUP, p.d, p.rot);
  const __nv_bfloat16* row = p.x + t * p.ld;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    if (i >= steps) break;
    const int h = h0 + i * HPW;
    const bool has = l.has && h < all;
    qk_ask(&mem[2 * i][threadIdx.x], has ? row + h * p.d + l.a : row, has);
    qk_ask(&mem[2 * i + 1][threadIdx.x], has ? row + h * p.d + l.b : row, has);
  }
  qk_commit();
  QkAngles angles;
  qk_angles<PAIRS>(p, l, t, angles);
  const float inv_d = 1.f / p.d;
  qk_wait<0>();
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    if (i >= steps) break;
    const int h = h0 + i * HPW, which = h >= p.heads[0];
    const bool has = l.has && h < all, weighted = has && p.w[which];
    uint4 wa, wb;
    if (weighted) {
      wa = *reinterpret_cast<const uint4*>(p.w[which] + l.a);
      wb = *reinterpret_cast<const uint4*>(p.w[which] + l.b);
    }
    QkPairs f = qk_unpack<PAIRS>(mem[2 * i][threadIdx.x], mem[2 * i + 1][threadIdx.x]);
    const float r = rsqrtf(qk_sum<GROUP>(qk_dot(f, f)) * inv_d + p.eps);
    const f32x2 rr = f2_pack(r, r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f.u[e] = f2_mul(f.u[e], rr);
      f.v[e] = f2_mul(f.v[e], rr);
    }
    if (weighted) f = qk_times(f, qk_unpack<PAIRS>(wa, wb));
    if (l.turned) qk_turn<false>(f, angles);
    if (has) {
      __nv_bfloat16* dst = p.y[which] + ((long long)t * p.heads[which] + (which ? h - p.heads[0] : h)) * p.d;
      qk_store<PAIRS>(f, dst + l.a, dst + l.b);
    }
  }
}

// A warp's way through one kind of heads: one block of a token's, every `stride`-th token.
struct QkWalk {
  int t, block, stride;
  __device__ __forceinline__ QkWalk(int blocks, int warp, int warps) {
    stride = warps / blocks;
    block = warp % blocks;
    t = warp / blocks < stride ? warp / blocks : 0x7fffffff;
  }
  __device__ __forceinline__ void next(int tokens) { t = t < tokens - stride ? t + stride : 0x7fffffff; }
};

// All queries, then all keys, in units of QB_STEPS x 32 / GROUP heads of a token, then the values' gradients as they are.
template <int GROUP, bool PAIRS, bool SUMS>
__global__ void __launch_bounds__(QK_THREADS, QB_CTAS)
qk_norm_bwd_kernel(const QkNorm p) {
  if (!chain_begin()) return;
  constexpr int HPW = 32 / GROUP, HEADS = QB_STEPS * HPW;
  extern __shared__ uint4 qk_mem[];          // [stages][steps][4][threads], then the warps' sums
  const int lane = threadIdx.x & 31, warp = warp_index(), group = lane / GROUP;
  const int me = blockIdx.x * QK_WARPS + warp, warps = gridDim.x * QK_WARPS;
  const QkLane l(lane % GROUP, p.d, p.rot);
  const int width = (p.heads[0] + 2 * p.heads[1]) * p.d;
  const float inv_d = 1.f / p.d;
  constexpr int VECS = QB_STEPS * 4;         // of a thread's to a stage
  const int v_vecs = p.heads[1] * p.d / 8;
  auto blocks_of = [&](int kind) { return kind < 2 ? (p.heads[kind] + HEADS - 1) / HEADS : (v_vecs + VECS * 32 - 1) / (VECS * 32); };
  auto place = [&](int stage, int i, int what) { return qk_mem + ((stage * QB_STEPS + i) * 4 + what) * QK_THREADS + threadIdx.x; };
  float* sums = reinterpret_cast<float*>(qk_mem + QB_STAGES * QB_STEPS * 4 * QK_THREADS);      // of queries, of keys: [warps][d]
  int kind = 0, ask_stage = 0, stage = 0;    // (kind: of the next unit to be asked for)
  QkWalk ahead(blocks_of(0), me, warps);
  auto ask = [&]() {                         // (a group each time, also behind the last unit)
    while (ahead.t >= p.tokens && kind < 2) ahead = QkWalk(blocks_of(++kind), me, warps);
    if (ahead.t < p.tokens && kind == 2) {
      const uint4* g = reinterpret_cast<const uint4*>(p.dy[2]) + (long long)ahead.t * v_vecs;
      const int at = ahead.block * VECS * 32 + lane;
#pragma unroll
      for (int i = 0; i < VECS; ++i) qk_ask(place(ask_stage, 0, i), g + (at + 32 * i < v_vecs ? at + 32 * i : 0), at + 32 * i < v_vecs);
      ahead.next(p.tokens);
    } else if (ahead.t < p.tokens) {
      const int n = p.heads[kind], h0 = ahead.block * HEADS + group;
      const __nv_bfloat16* x = p.x + ahead.t * p.ld + (kind ? p.heads[0] : 0) * p.d;
      const __nv_bfloat16* g = p.dy[kind] + (long long)ahead.t * n * p.d;
#pragma unroll
      for (int i = 0; i < QB_STEPS; ++i) {
        const int h = h0 + i * HPW;
        const bool has = l.has && h < n;
        const int a = has ? h * p.d + l.a : 0, b = has ? h * p.d + l.b : 0;
        qk_ask(place(ask_stage, i, 0), x + a, has);
        qk_ask(place(ask_stage, i, 1), x + b, has);
        qk_ask(place(ask_stage, i, 2), g + a, has);
        qk_ask(place(ask_stage, i, 3), g + b, has);
      }
      ahead.next(p.tokens);
    }
    qk_commit();
    if (++ask_stage == QB_STAGES) ask_stage = 0;
  };
#pragma unroll
  for (int i = 0; i < QB_STAGES; ++i) ask();
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int n = p.heads[which];
    uint4 wa = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u), wb = wa;      // ones
    if (p.w[which] && l.has) {
      wa = *reinterpret_cast<const uint4*>(p.w[which] + l.a);
      wb = *reinterpret_cast<const uint4*>(p.w[which] + l.b);
    }
    const QkPairs w = qk_unpack<PAIRS>(wa, wb);
    QkPairs acc;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc.u[e] = acc.v[e] = f2_pack(0.f, 0.f);
#pragma unroll 1
    for (QkWalk at(blocks_of(which), me, warps); at.t < p.tokens; at.next(p.tokens)) {
      QkAngles angles;
      qk_angles<PAIRS>(p, l, at.t, angles);
      const int left = min(HEADS, n - at.block * HEADS);
      __nv_bfloat16* dst = p.dx + (long long)at.t * width + ((which ? p.heads[0] : 0) + at.block * HEADS + group) * p.d;
      qk_wait<QB_STAGES - 1>();
#pragma unroll
      for (int i = 0; i < QB_STEPS; ++i) {
        if (i * HPW >= left) break;
        QkPairs g = qk_unpack<PAIRS>(*place(stage, i, 2), *place(stage, i, 3));
        if (l.turned) qk_turn<true>(g, angles);
        const QkPairs x = qk_unpack<PAIRS>(*place(stage, i, 0), *place(stage, i, 1));
        float dot;
        QkPairs gx;
        if (SUMS) {
          gx = qk_times(g, x);
          dot = qk_dot(gx, w);
          g = qk_times(g, w);
        } else {
          g = qk_times(g, w);
          dot = qk_dot(g, x);
        }
        const float r = rsqrtf(qk_sum<GROUP>(qk_dot(x, x)) * inv_d + p.eps), k = -r * (r * (r * (qk_sum<GROUP>(dot) * inv_d)));      // (r^3 may overflow)
        const f32x2 rr = f2_pack(r, r), kk = f2_pack(k, k);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (SUMS) {                        // (a lane without a head adds zeros)
            acc.u[e] = f2_fma(gx.u[e], rr, acc.u[e]);
            acc.v[e] = f2_fma(gx.v[e], rr, acc.v[e]);
          }
          g.u[e] = f2_fma(x.u[e], kk, f2_mul(g.u[e], rr));
          g.v[e] = f2_fma(x.v[e], kk, f2_mul(g.v[e], rr));
        }
        if (l.has && i * HPW + group < left) qk_store<PAIRS>(g, dst + i * HPW * p.d + l.a, dst + i * HPW * p.d + l.b);
      }
      ask();
      if (++stage == QB_STAGES) stage = 0;
    }
    if (SUMS) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[4];                          // columns of u[e], then of v[e]
        f2_unpack(acc.u[e], f[0], f[1]);
        f2_unpack(acc.v[e], f[2], f[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int o = GROUP; o < 32; o <<= 1) f[i] += __shfl_xor_sync(0xffffffffu, f[i], o);
        if (lane < GROUP && l.has) {
          float* to = sums + (which * QK_WARPS + warp) * p.d + (PAIRS && e >= 2 ? l.b + 4 * (e - 2) : l.a + (PAIRS ? 4 * e : 2 * e));
          if (PAIRS) {
            to[0] = f[0]; to[2] = f[1];
            to[1] = f[2]; to[3] = f[3];
          } else {
            to[0] = f[0]; to[1] = f[1];
            to[l.b - l.a] = f[2]; to[l.b - l.a + 1] = f[3];
          }
        }
      }
    }
  }
#pragma unroll 1
  for (QkWalk at(blocks_of(2), me, warps); at.t < p.tokens; at.next(p.tokens)) {
    uint4* dst = reinterpret_cast<uint4*>(p.dx + (long long)at.t * width + (p.heads[0] + p.heads[1]) * p.d);
    const int first = at.block * VECS * 32 + lane;
    qk_wait<QB_STAGES - 1>();
#pragma unroll
    for (int i = 0; i < VECS; ++i)
      if (first + 32 * i < v_vecs) dst[first + 32 * i] = *place(stage, 0, i);
    ask();
    if (++stage == QB_STAGES) stage = 0;
  }
  if (SUMS) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * p.d; i += QK_THREADS) {
      const float* from = sums + (i < p.d ? i : i + (QK_WARPS - 1) * p.d);
      float a = from[0];
#pragma unroll
      for (int w = 1; w < QK_WARPS; ++w) a += from[w * p.d];
      p.parts[(long long)blockIdx.x * 2 * p.d + i] = a;
    }
  }
}

// dw[which][c] = sum of the CTAs' parts; in fp32 and, where there is a place for it, rounded.  A CTA takes 32 columns, 32 parts at a time:
// a thread has up to ten of the 296, which are all asked for at once.
constexpr int QD_ROWS = 32, QD_AHEAD = 10;
__global__ void __launch_bounds__(QD_ROWS * 32)
qk_norm_dw_kernel(const float* __restrict__ parts, float* __restrict__ dw, __nv_bfloat16* dwq, __nv_bfloat16* dwk, int n, int d) {
  if (!chain_begin()) return;
  __shared__ float sums[QD_ROWS][32];
  const int lane = threadIdx.x & 31, row0 = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, which = blockIdx.y;
  float a = 0.f;
  for (int r0 = row0; r0 < n; r0 += QD_ROWS * QD_AHEAD) {
    float v[QD_AHEAD];
#pragma unroll
    for (int i = 0; i < QD_AHEAD; ++i)
      v[i] = r0 + QD_ROWS * i < n && col < d ? parts[((long long)(r0 + QD_ROWS * i) * 2 + which) * d + col] : 0.f;
#pragma unroll
    for (int i = 0; i < QD_AHEAD; ++i) a += v[i];
  }
  sums[row0][lane] = a;
  __syncthreads();
  if (row0 != 0 || col >= d) return;
#pragma unroll
  for (int r = 1; r < QD_ROWS; ++r) a += sums[r][lane];
  dw[which * d + col] = a;
  __nv_bfloat16* out = which ? dwk : dwq;
  if (out) out[col] = __float2bfloat16(a);
}

static int qk_group(int d) {
  int g = 1;
  while (g * 16 < d) g *= 2;
  return g;
}

// More shared memory than a launch has by itself, once for each device.
template <typename F>
static cudaError_t qk_allow(F* f, int smem, std::atomic<unsigned>& ready) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device > 31 || !(ready.load(std::memory_order_relaxed) >> device & 1))) {
    e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && device <= 31) ready.fetch_or(1u << device, std::memory_order_relaxed);
  }
  return e;
}

// CTAs for units of so many heads: a warp for each unit as far as they go.
static int qk_grid(const QkNorm& p, int unit_heads, int most) {
  const long long units = (long long)p.tokens * ((p.heads[0] + unit_heads - 1) / unit_heads + (p.heads[1] + unit_heads - 1) / unit_heads);
  const long long need = (units + QK_WARPS - 1) / QK_WARPS;
  return (int)(need < most ? need : most);
}

static int qk_bwd_grid(const QkNorm& p) { return qk_grid(p, QB_STEPS * (32 / qk_group(p.d)), QB_CTAS * sm_count()); }

template <int GROUP, bool PAIRS, int STEPS>
static cudaError_t launch_qk_fwd(const QkNorm& p, cudaStream_t stream) {
  const unsigned steps = (p.heads[0] + p.heads[1] + 32 / GROUP - 1) / (32 / GROUP), blocks = (steps + STEPS - 1) / STEPS;
  const unsigned units = blocks * p.tokens;
  return chain(qk_norm_fwd_kernel<GROUP, PAIRS, STEPS>, (units + QK_WARPS - 1) / QK_WARPS, QK_THREADS, 0, stream, p, units, blocks,
               (int)((steps + blocks - 1) / blocks));
}
template <int GROUP, bool PAIRS>
static cudaError_t launch_qk_fwd(const QkNorm& p, cudaStream_t stream) {
  // Few heads in all: two steps to a warp, for more warps; else up to five, for more under way.  us, 2 / 5: 48 tokens of 32 / 8 heads 2.3 / 3.5,
  // 2103 of 16 / 4 of 64 columns 3.8 / 4.9, 2049 of 40 / 8 9.9 / 9.9; 8192 of 32 / 8 30.8 / 28.8, 32768 of 64 / 8 202 / 179.
  const long long steps = (p.heads[0] + p.heads[1] + 32 / GROUP - 1) / (32 / GROUP);
  return steps * p.tokens < 64LL * QK_WARPS * sm_count() ? launch_qk_fwd<GROUP, PAIRS, 2>(p, stream) : launch_qk_fwd<GROUP, PAIRS, 5>(p, stream);
}

template <int GROUP, bool PAIRS, bool SUMS>
static cudaError_t launch_qk_bwd(const QkNorm& p, cudaStream_t stream) {
  const int smem = QB_STAGES * QB_STEPS * 4 * QK_THREADS * 16 + (SUMS ? 2 * QK_WARPS * GROUP * 16 * 4 : 0);
  static std::atomic<unsigned> ready{0};
  const cudaError_t e = qk_allow(qk_norm_bwd_kernel<GROUP, PAIRS, SUMS>, smem, ready);
  if (e != cudaSuccess) return e;
  return chain(qk_norm_bwd_kernel<GROUP, PAIRS, SUMS>, qk_bwd_grid(p), QK_THREADS, smem, stream, p);
}
template <int GROUP, bool PAIRS>
static cudaError_t launch_qk_bwd(const QkNorm& p, bool sums, cudaStream_t stream) {
  return sums ? launch_qk_bwd<GROUP, PAIRS, true>(p, stream) : launch_qk_bwd<GROUP, PAIRS, false>(p, stream);
}

static bool qk_sizes_ok(const QkNorm& p) {
  const long long most = 0x7fffffffLL;
  return p.tokens >= 0 && p.heads[0] >= 1 && p.heads[1] >= 1 && p.heads[0] <= 1024 && p.heads[1] <= 1024 && p.d >= 16 && p.d <= 512 && p.d % 16 == 0 && p.rot >= 0 && p.rot <= p.d &&
         p.rot % 16 == 0 && p.ld % 8 == 0 && (p.pos || p.seq > 0) && p.table > 0 && (p.pos || p.seq <= p.table) &&
         (long long)(p.heads[0] + 2LL * p.heads[1]) * p.d <= most && (long long)p.tokens * (p.heads[0] + p.heads[1]) <= most;
}
static bool qk_aligned(std::initializer_list<const void*> ps) {
  for (const void* a : ps)
    if (reinterpret_cast<uintptr_t>(a) % 16) return false;
  return true;
}

#define QK_GROUPS(CALL)                                                                                                       \
  switch (qk_group(p.d)) {                                                                                                    \
    case 1: launched = CALL(1); break;                                                                                                   \
    case 2: launched = CALL(2); break;                                                                                                   \
    case 4: launched = CALL(4); break;                                                                                                   \
    case 8: launched = CALL(8); break;                                                                                                   \
    case 16: launched = CALL(16); break;                                                                                                 \
    default: launched = CALL(32); break;                                                                                                 \
  }

}  // namespace tpb

using namespace tpb;

// x [tokens, (hq + 2 hkv) * d] bf16, rows ld apart: q [tokens, hq, d] and k [tokens, hkv, d] get the normalised and rotated heads.
// wq, wk [d] bf16 or null; cos, sin fp32 [table, rot / 2]; pos int32 [tokens] or null (token % seq).  interleaved: pairs of neighbours.
// All pointers but pos 16-byte aligned.
extern "C" int tpb_qk_norm_fwd(const void* x, long long ld, const void* wq, const void* wk, const float* cos, const float* sin, int table,
                               const int* pos, int seq, void* q, void* k, int tokens, int hq, int hkv, int d, int rot, float eps,
                               int interleaved, void* stream) {
  QkNorm p = {};
  p.x = static_cast<const __nv_bfloat16*>(x); p.ld = ld;
  p.w[0] = static_cast<const __nv_bfloat16*>(wq); p.w[1] = static_cast<const __nv_bfloat16*>(wk);
  p.cos = cos; p.sin = sin; p.table = table; p.pos = pos; p.seq = seq;
  p.y[0] = static_cast<__nv_bfloat16*>(q); p.y[1] = static_cast<__nv_bfloat16*>(k);
  p.tokens = tokens; p.heads[0] = hq; p.heads[1] = hkv; p.d = d; p.rot = rot; p.eps = eps;
  p.status = status_block();
  if (!qk_sizes_ok(p) || !qk_aligned({x, wq, wk, cos, sin, q, k})) return -2;
  if (tokens == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t launched = cudaSuccess;
#define QK_CALL(G) (interleaved ? launch_qk_fwd<G, true>(p, st) : launch_qk_fwd<G, false>(p, st))
  QK_GROUPS(QK_CALL)
#undef QK_CALL
  const cudaError_t e = launched != cudaSuccess ? launched : cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

// Floats of scratch for the weights' gradients: [2][d] sums in front, then the CTAs' parts.
extern "C" long long tpb_qk_norm_bwd_scratch(int tokens, int d) {
  return tokens > 0 ? 2LL * d * (1 + QB_CTAS * sm_count()) : 2LL * d;
}

// Gradients of the above: dx [tokens, (hq + 2 hkv) * d] from dq, dk and dv (contiguous; dv's columns are copied).  sums: scratch
// of tpb_qk_norm_bwd_scratch floats, whose first [2][d] become the weights' gradients, or null; dwq, dwk: the same in bf16, or null.
extern "C" int tpb_qk_norm_bwd(const void* x, long long ld, const void* wq, const void* wk, const float* cos, const float* sin, int table,
                               const int* pos, int seq, const void* dq, const void* dk, const void* dv, void* dx, float* sums, void* dwq,
                               void* dwk, int tokens, int hq, int hkv, int d, int rot, float eps, int interleaved, void* stream) {
  QkNorm p = {};
  p.x = static_cast<const __nv_bfloat16*>(x); p.ld = ld;
  p.w[0] = static_cast<const __nv_bfloat16*>(wq); p.w[1] = static_cast<const __nv_bfloat16*>(wk);
  p.cos = cos; p.sin = sin; p.table = table; p.pos = pos; p.seq = seq;
  p.dy[0] = static_cast<const __nv_bfloat16*>(dq); p.dy[1] = static_cast<const __nv_bfloat16*>(dk);
  p.dy[2] = static_cast<const __nv_bfloat16*>(dv); p.dx = static_cast<__nv_bfloat16*>(dx);
  p.parts = sums ? sums + 2 * d : nullptr;
  p.tokens = tokens; p.heads[0] = hq; p.heads[1] = hkv; p.d = d; p.rot = rot; p.eps = eps;
  p.status = status_block();
  if (!qk_sizes_ok(p) || !qk_aligned({x, wq, wk, cos, sin, dq, dk, dv, dx})) return -2;
  if (tokens == 0 && !sums) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = qk_bwd_grid(p);
  cudaError_t launched = cudaSuccess;
  if (tokens > 0) {
#define QK_CALL(G) (interleaved ? launch_qk_bwd<G, true>(p, sums != nullptr, st) : launch_qk_bwd<G, false>(p, sums != nullptr, st))
    QK_GROUPS(QK_CALL)
#undef QK_CALL
  }
  if (sums && launched == cudaSuccess)
    chain(qk_norm_dw_kernel, dim3((d + 31) / 32, 2), QD_ROWS * 32, 0, st, (const float*)p.parts, sums, static_cast<__nv_bfloat16*>(dwq),
          static_cast<__nv_bfloat16*>(dwk), tokens > 0 ? grid : 0, d);
  const cudaError_t e = launched != cudaSuccess ? launched : cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
