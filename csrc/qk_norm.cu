// Norms of the query and key heads of a fused projection with the position rotation in the same pass, and their gradient.
//
//   y = R(p) (w * x r),  r = (mean(x^2) + eps)^-1/2 over the d columns of a head;  w optional;  R(p) turns pairs of the leading
//   `rot` columns by the angles of position p: columns (i, i + rot / 2), or neighbours (2i, 2i + 1);
//   g = R(p)^T dy,  dw = sum over tokens and heads of g x r,  dx = r w g - x r^3 mean(w g x).
//
// A head is read once and written once, three bf16 numbers in and out for each product, so memory bounds both directions.  A lane
// holds two 16-byte vectors of a head, the two that are turned with one another: the rotation needs no neighbour, and the sums of a
// head of 128 columns are three shuffles over eight lanes.  Statistics, products and sums are fp32; results are rounded once.  The
// gradient takes r from x again (x has to be read there anyway) and, of the weights, adds up in registers over all heads that a
// thread sees, then over the CTA's warps and over the CTAs, in an order that only the sizes decide.

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

__device__ __forceinline__ void qk_unpack(const uint4& u, float* f) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
}
__device__ __forceinline__ uint4 qk_pack(const float* f) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

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

// cos and sin of a lane's eight pairs.
template <bool PAIRS>
__device__ __forceinline__ void qk_angles(const QkNorm& p, const QkLane& l, int t, float* c, float* s) {
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
  c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
  s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
}

// f: the first vector's eight numbers, then the second's.
template <bool PAIRS, bool BACK>
__device__ __forceinline__ void qk_turn(float* f, const float* c, const float* s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float& u = f[PAIRS ? 2 * i : i];
    float& v = f[PAIRS ? 2 * i + 1 : i + 8];
    const float sn = BACK ? -s[i] : s[i], x = u * c[i] - v * sn, y = v * c[i] + u * sn;
    u = x;
    v = y;
  }
}

template <int GROUP>
__device__ __forceinline__ float qk_sum(float v) {
#pragma unroll
  for (int o = 1; o < GROUP; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A warp takes STEPS x 32 / GROUP heads of a token.
template <int GROUP, bool PAIRS, int STEPS>
__global__ void __launch_bounds__(QK_THREADS)
qk_norm_fwd_kernel(const QkNorm p, unsigned units, unsigned blocks) {
  if (!chain_begin()) return;
  constexpr int HPW = 32 / GROUP;
  const unsigned unit = blockIdx.x * QK_WARPS + warp_index();
  if (unit >= units) return;
  const int lane = threadIdx.x & 31, t = unit / blocks, h0 = (unit % blocks) * STEPS * HPW + lane / GROUP;
  const QkLane l(lane % GROUP, p.d, p.rot);
  const int all = p.heads[0] + p.heads[1];
  const __nv_bfloat16* row = p.x + t * p.ld;
  uint4 va[STEPS], vb[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int h = h0 + i * HPW;
    va[i] = vb[i] = make_uint4(0, 0, 0, 0);
    if (l.has && h < all) {
      va[i] = *reinterpret_cast<const uint4*>(row + h * p.d + l.a);
      vb[i] = *reinterpret_cast<const uint4*>(row + h * p.d + l.b);
    }
  }
  float c[8], s[8];
  qk_angles<PAIRS>(p, l, t, c, s);
  const float inv_d = 1.f / p.d;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int h = h0 + i * HPW;
    float f[16], sq = 0.f;
    qk_unpack(va[i], f);
    qk_unpack(vb[i], f + 8);
#pragma unroll
    for (int e = 0; e < 16; ++e) sq = fmaf(f[e], f[e], sq);
    const float r = rsqrtf(qk_sum<GROUP>(sq) * inv_d + p.eps);
    if (!l.has || h >= all) continue;
    const int which = h >= p.heads[0];
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e] = mul_exact(f[e], r);
    if (p.w[which]) {
      float w[16];
      qk_unpack(*reinterpret_cast<const uint4*>(p.w[which] + l.a), w);
      qk_unpack(*reinterpret_cast<const uint4*>(p.w[which] + l.b), w + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] *= w[e];
    }
    if (l.turned) qk_turn<PAIRS, false>(f, c, s);
    const int hh = which ? h - p.heads[0] : h;
    __nv_bfloat16* dst = p.y[which] + ((long long)t * p.heads[which] + hh) * p.d;
    *reinterpret_cast<uint4*>(dst + l.a) = qk_pack(f);
    *reinterpret_cast<uint4*>(dst + l.b) = qk_pack(f + 8);
  }
}

// All queries, then all keys, then the values' gradients as they are; each in units of STEPS x 32 / GROUP heads of a token.
template <int GROUP, bool PAIRS, bool SUMS, int STEPS>
__global__ void __launch_bounds__(QK_THREADS, 2)
qk_norm_bwd_kernel(const QkNorm p) {
  if (!chain_begin()) return;
  constexpr int HPW = 32 / GROUP;
  __shared__ float sums[QK_WARPS][512];
  const int warp = warp_index(), lane = threadIdx.x & 31, group = lane / GROUP;
  const unsigned first = blockIdx.x * QK_WARPS + warp, stride = gridDim.x * QK_WARPS;
  const QkLane l(lane % GROUP, p.d, p.rot);
  const long long width = (long long)(p.heads[0] + 2 * p.heads[1]) * p.d;
  const float inv_d = 1.f / p.d;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int n = p.heads[which], head0 = which ? p.heads[0] : 0;
    const unsigned blocks = (n + STEPS * HPW - 1) / (STEPS * HPW), units = blocks * p.tokens;
    uint4 wa = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u), wb = wa;      // ones
    if (p.w[which] && l.has) {
      wa = *reinterpret_cast<const uint4*>(p.w[which] + l.a);
      wb = *reinterpret_cast<const uint4*>(p.w[which] + l.b);
    }
    float acc[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll 1
    for (unsigned unit = first; unit < units; unit += stride) {
      const int t = unit / blocks, h0 = (unit % blocks) * STEPS * HPW + group;
      const __nv_bfloat16* xr = p.x + t * p.ld + head0 * p.d;
      const __nv_bfloat16* gr = p.dy[which] + (long long)t * n * p.d;
      __nv_bfloat16* dr = p.dx + t * width + head0 * p.d;
      uint4 v[STEPS][4];
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int h = h0 + i * HPW;
        v[i][0] = v[i][1] = v[i][2] = v[i][3] = make_uint4(0, 0, 0, 0);
        if (l.has && h < n) {
          v[i][0] = *reinterpret_cast<const uint4*>(xr + h * p.d + l.a);
          v[i][1] = *reinterpret_cast<const uint4*>(xr + h * p.d + l.b);
          v[i][2] = *reinterpret_cast<const uint4*>(gr + h * p.d + l.a);
          v[i][3] = *reinterpret_cast<const uint4*>(gr + h * p.d + l.b);
        }
      }
      float c[8], s[8];
      qk_angles<PAIRS>(p, l, t, c, s);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int h = h0 + i * HPW;
        float x[16], g[16], w[16], sq = 0.f, dot = 0.f;
        qk_unpack(v[i][0], x);
        qk_unpack(v[i][1], x + 8);
        qk_unpack(v[i][2], g);
        qk_unpack(v[i][3], g + 8);
        if (l.turned) qk_turn<PAIRS, true>(g, c, s);
        qk_unpack(wa, w);
        qk_unpack(wb, w + 8);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          sq = fmaf(x[e], x[e], sq);
          dot = fmaf(g[e] * w[e], x[e], dot);
        }
        sq = qk_sum<GROUP>(sq);
        dot = qk_sum<GROUP>(dot);
        const float r = rsqrtf(sq * inv_d + p.eps), k = r * r * (dot * inv_d);
        if (!l.has || h >= n) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (SUMS) acc[e] = fmaf(g[e], mul_exact(x[e], r), acc[e]);
          g[e] = r * (g[e] * w[e] - x[e] * k);
        }
        *reinterpret_cast<uint4*>(dr + h * p.d + l.a) = qk_pack(g);
        *reinterpret_cast<uint4*>(dr + h * p.d + l.b) = qk_pack(g + 8);
      }
    }
    if (SUMS) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int o = GROUP; o < 32; o <<= 1) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
      __syncthreads();
      if (lane < GROUP && l.has) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sums[warp][l.a + e] = acc[e];
          sums[warp][l.b + e] = acc[8 + e];
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < p.d; i += QK_THREADS) {
        float a = sums[0][i];
#pragma unroll
        for (int w = 1; w < QK_WARPS; ++w) a += sums[w][i];
        p.parts[((long long)blockIdx.x * 2 + which) * p.d + i] = a;
      }
    }
  }
  const int vecs = p.heads[1] * p.d / 8;
  const long long off = (long long)(p.heads[0] + p.heads[1]) * p.d;
  for (unsigned t = first; t < (unsigned)p.tokens; t += stride) {
    const uint4* src = reinterpret_cast<const uint4*>(p.dy[2]) + (long long)t * vecs;
    uint4* dst = reinterpret_cast<uint4*>(p.dx + t * width + off);
#pragma unroll 4
    for (int i = lane; i < vecs; i += 32) dst[i] = src[i];
  }
}

// dw[which][c] = sum of the CTAs' parts; in fp32 and, where there is a place for it, rounded.  A CTA takes 32 columns.
__global__ void __launch_bounds__(256)
qk_norm_dw_kernel(const float* __restrict__ parts, float* __restrict__ dw, __nv_bfloat16* dwq, __nv_bfloat16* dwk, int n, int d) {
  if (!chain_begin()) return;
  __shared__ float sums[8][32];
  const int lane = threadIdx.x & 31, row0 = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, which = blockIdx.y;
  float a = 0.f;
  if (col < d)
#pragma unroll 8
    for (int r = row0; r < n; r += 8) a += parts[((long long)r * 2 + which) * d + col];
  sums[row0][lane] = a;
  __syncthreads();
  if (row0 != 0 || col >= d) return;
#pragma unroll
  for (int r = 1; r < 8; ++r) a += sums[r][lane];
  dw[which * d + col] = a;
  __nv_bfloat16* out = which ? dwk : dwq;
  if (out) out[col] = __float2bfloat16(a);
}

static int qk_group(int d) {
  int g = 1;
  while (g * 16 < d) g *= 2;
  return g;
}

template <int GROUP, bool PAIRS>
static void launch_qk_fwd(const QkNorm& p, cudaStream_t stream) {
  constexpr int STEPS = 4;
  const unsigned all = p.heads[0] + p.heads[1], per = STEPS * (32 / GROUP), blocks = (all + per - 1) / per, units = blocks * p.tokens;
  chain(qk_norm_fwd_kernel<GROUP, PAIRS, STEPS>, (units + QK_WARPS - 1) / QK_WARPS, QK_THREADS, 0, stream, p, units, blocks);
}

static int qk_bwd_grid(int tokens) {
  const int most = 2 * sm_count();
  return (tokens + 1) / 2 < most ? (tokens + 1) / 2 : most;
}

template <int GROUP, bool PAIRS>
static void launch_qk_bwd(const QkNorm& p, bool sums, cudaStream_t stream) {
  constexpr int STEPS = 2;
  const int grid = qk_bwd_grid(p.tokens);
  if (sums) chain(qk_norm_bwd_kernel<GROUP, PAIRS, true, STEPS>, grid, QK_THREADS, 0, stream, p);
  else chain(qk_norm_bwd_kernel<GROUP, PAIRS, false, STEPS>, grid, QK_THREADS, 0, stream, p);
}

static bool qk_sizes_ok(const QkNorm& p) {
  const long long most = 0x7fffffffLL;
  return p.tokens >= 0 && p.heads[0] >= 1 && p.heads[1] >= 1 && p.d >= 16 && p.d <= 512 && p.d % 16 == 0 && p.rot >= 0 && p.rot <= p.d &&
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
    case 1: CALL(1); break;                                                                                                   \
    case 2: CALL(2); break;                                                                                                   \
    case 4: CALL(4); break;                                                                                                   \
    case 8: CALL(8); break;                                                                                                   \
    case 16: CALL(16); break;                                                                                                 \
    default: CALL(32); break;                                                                                                 \
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
#define QK_CALL(G) (interleaved ? launch_qk_fwd<G, true>(p, st) : launch_qk_fwd<G, false>(p, st))
  QK_GROUPS(QK_CALL)
#undef QK_CALL
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

// Floats of scratch for the weights' gradients: [2][d] sums in front, then the CTAs' parts.
extern "C" long long tpb_qk_norm_bwd_scratch(int tokens, int d) { return 2LL * d * (1 + qk_bwd_grid(tokens)); }

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
  const int grid = qk_bwd_grid(tokens);
  if (tokens > 0) {
#define QK_CALL(G) (interleaved ? launch_qk_bwd<G, true>(p, sums != nullptr, st) : launch_qk_bwd<G, false>(p, sums != nullptr, st))
    QK_GROUPS(QK_CALL)
#undef QK_CALL
  }
  if (sums)
    chain(qk_norm_dw_kernel, dim3((d + 31) / 32, 2), 256, 0, st, (const float*)p.parts, sums, static_cast<__nv_bfloat16*>(dwq),
          static_cast<__nv_bfloat16*>(dwk), tokens > 0 ? grid : 0, d);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
