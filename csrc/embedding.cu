// Embedding: rows of a table, scaled, and the table's gradient by sorted tokens.
//
//   out[t] = scale * E[id[t]],   dE[v] (+)= scale * sum of dout[t] over the tokens t with id[t] = v, in ascending order of t.
//
// Both are bound by memory.  The gradient of a training step writes the whole table (most rows as zeros) and reads dout once;
// what makes it slow otherwise are atomics, which read and write an fp32 table that has to be zeroed before and rounded behind, in an
// order that differs from run to run.  Here three kernels give every row one writer:
//
// * embedding_plan_kernel puts the tokens in order of their ids.  A CTA has a range of ids and looks at all tokens, so no CTA has to
//   wait for another: its 32 warps count what each id has in their parts of the tokens, the counts become places (how many
//   tokens have ids in front of the range is counted on the way), and a second look puts the tokens there, in order.
// * embedding_sum_kernel cuts that order into chunks of equal size, whatever the ids: a warp adds up 256 columns of a chunk's rows
//   in fp32.  An id whose tokens lie within a chunk is written at once; one that reaches over a chunk's border leaves its part, at most
//   two a chunk.  Rows without a token become zeros, between the chunks' loads.
// * embedding_join_kernel adds up the parts, in the chunks' order; many of them (the padding's row) are shared by a CTA's warps.

#include <atomic>

#include "common.cuh"
#include "tpb.h"

namespace tpb {

int sm_count();

constexpr int EP_WARPS = 32;                 // of the planning kernel
constexpr int EP_ROWS = 1024;                // most ids to a CTA of it
constexpr int EJ_WARPS = 32;                 // of the joining kernel
constexpr int EJ_LONG = 16;                  // parts from which a CTA's warps share an id

__device__ __forceinline__ void emb_unpack(const uint4& u, float* f) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
}
__device__ __forceinline__ uint4 emb_pack(const float* f) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

// A warp takes up to 4 x 32 vectors of a token's row.
template <bool SCALED>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const uint4* __restrict__ table, const long long* __restrict__ ids, uint4* __restrict__ out, unsigned units,
                     unsigned blocks, int nvec, long long vocab, long long row0, float scale) {
  if (!chain_begin()) return;
  const unsigned unit = blockIdx.x * 8 + warp_index();
  if (unit >= units) return;
  const unsigned t = unit / blocks;
  const int v0 = (unit % blocks) * 128 + (threadIdx.x & 31);
  const long long id = ids[t] - row0;
  const bool in = id >= 0 && id < vocab;
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = in && v0 + 32 * i < nvec ? table[id * nvec + v0 + 32 * i] : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (v0 + 32 * i >= nvec) break;
    if (SCALED) {
      float f[8];
      emb_unpack(v[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = mul_exact(f[e], scale);
      v[i] = emb_pack(f);
    }
    out[(long long)t * nvec + v0 + 32 * i] = v[i];
  }
}

// Scratch of the gradient, in this order: range [rows] (first place, tokens), order [tokens], sorted ids [tokens], number of tokens
// that have a row [1], parts.
struct EmbGrad {
  const long long* ids;
  const __nv_bfloat16* dout;
  void* dtable;
  int2* range;
  int *order, *sorted, *valid;
  float* part;                               // [chunks][2][dim]: of the id that began before the chunk, of the one that goes on behind it
  long long row0;
  int tokens, rows, dim, chunk, chunks, per;  // per: ids to a CTA of the planning kernel
  float scale;
};

__global__ void __launch_bounds__(EP_WARPS * 32)
embedding_plan_kernel(const EmbGrad p) {
  if (!chain_begin()) return;
  extern __shared__ int ep_hist[];           // [warps][per]
  __shared__ int s_warp[EP_WARPS], s_below;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const long long first = p.row0 + (long long)blockIdx.x * p.per;
  const int mine = min(p.per, p.rows - (int)blockIdx.x * p.per);
  const int share = ((p.tokens + EP_WARPS * 32 - 1) / (EP_WARPS * 32)) * 32;
  const int t0 = min(warp * share, p.tokens), t1 = min(t0 + share, p.tokens);
  int* hist = ep_hist + warp * p.per;
  for (int i = threadIdx.x; i < EP_WARPS * p.per; i += EP_WARPS * 32) ep_hist[i] = 0;
  if (threadIdx.x == 0) s_below = 0;
  __syncthreads();
  // ---- how many tokens each id has in each warp's part, and how many have ids in front of this CTA's
  int below = 0;
#pragma unroll 8
  for (int t = t0 + lane; t < t1; t += 32) {
    const long long id = p.ids[t] - first;
    if (id >= 0 && id < mine) atomicAdd(&hist[id], 1);
    below += id < 0 && id >= p.row0 - first;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) below += __shfl_xor_sync(0xffffffffu, below, o);
  if (lane == 0 && below) atomicAdd(&s_below, below);
  __syncthreads();
  // ---- their places: a thread for each id
  const int r = threadIdx.x;
  int count = 0;
  if (r < mine)
    for (int w = 0; w < EP_WARPS; ++w) {
      const int n = ep_hist[w * p.per + r];
      ep_hist[w * p.per + r] = count;
      count += n;
    }
  int sum = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) s_warp[warp] = sum;
  __syncthreads();
  int start = s_below + sum - count;
  for (int w = 0; w < warp; ++w) start += s_warp[w];
  if (r < mine) {
    for (int w = 0; w < EP_WARPS; ++w) ep_hist[w * p.per + r] += start;
    p.range[blockIdx.x * p.per + r] = make_int2(start, count);
    if (blockIdx.x * p.per + r == p.rows - 1) *p.valid = start + count;
  }
  __syncthreads();
  // ---- the tokens, in order: those of one id in a warp's 32 by lane
  for (int t = t0; t < t1; t += 32) {
    const long long id = t + lane < t1 ? p.ids[t + lane] - first : -1;
    const bool in = id >= 0 && id < mine;
    const unsigned any = __ballot_sync(0xffffffffu, in);
    if (any == 0) continue;
    if (in) {
      const unsigned same = __match_any_sync(any, (int)id);
      const int at = hist[id] + __popc(same & ((1u << lane) - 1));
      p.order[at] = t + lane;
      p.sorted[at] = blockIdx.x * p.per + (int)id;
      __syncwarp(any);
      if ((same & ((1u << lane) - 1)) == 0) hist[id] = at + __popc(same);
    }
    __syncwarp();
  }
}

template <bool F32>
__device__ __forceinline__ void emb_store(void* dtable, long long at, const float* acc, float scale, bool add) {
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = mul_exact(acc[e], scale);
  if (F32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(dtable) + at);
    float4 a = make_float4(f[0], f[1], f[2], f[3]), b = make_float4(f[4], f[5], f[6], f[7]);
    if (add) {
      const float4 x = dst[0], y = dst[1];
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
    }
    dst[0] = a;
    dst[1] = b;
  } else {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(dtable) + at);
    if (add) {
      float x[8];
      emb_unpack(*dst, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += x[e];
    }
    *dst = emb_pack(f);
  }
}

constexpr int ES_ZERO = 4;       // rows of a warp's look for ones without tokens

template <bool F32, bool ADD>
__global__ void __launch_bounds__(256)
embedding_sum_kernel(const EmbGrad p) {
  if (!chain_begin()) return;
  const int lane = threadIdx.x & 31, blocks = (p.dim + 255) / 256;
  const long long warp = blockIdx.x * 8LL + warp_index(), stride = gridDim.x * 8LL;
  const int valid = *p.valid;
  const long long items = (long long)((valid + p.chunk - 1) / p.chunk) * blocks;
  for (long long item = warp; item < items; item += stride) {
    const int c = (int)(item / blocks), col = (int)(item % blocks) * 256 + lane * 8, base = c * p.chunk;
    const int n = min(p.chunk, valid - base);
    const bool has = col < p.dim;
    const int before = base > 0 ? p.sorted[base - 1] : -1;
    float acc[8] = {};
    bool first = true;                       // the id of the chunk's first token
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int m = min(32, n - i0), at = base + i0 + lane;
      const int tok = lane < m ? p.order[at] : 0, id = lane < m ? p.sorted[at] : -1;
      const int next = lane < m && at + 1 < valid ? p.sorted[at + 1] : -1;
      const unsigned ends = __ballot_sync(0xffffffffu, lane < m && (id != next || i0 + lane == n - 1));
      const unsigned goes = __ballot_sync(0xffffffffu, id == next);
      for (int j0 = 0; j0 < m; j0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = __shfl_sync(0xffffffffu, tok, j0 + j);
          v[j] = has && j0 + j < m ? *reinterpret_cast<const uint4*>(p.dout + (long long)t * p.dim + col) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j0 + j >= m) break;
          float x[8];
          emb_unpack(v[j], x);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += x[e];
          if (ends >> (j0 + j) & 1) {
            const int run = __shfl_sync(0xffffffffu, id, j0 + j);
            const bool began = first && run == before, on = goes >> (j0 + j) & 1;
            if (has) {
              if (!began && !on) {
                emb_store<F32>(p.dtable, (long long)run * p.dim + col, acc, p.scale, ADD);
              } else {
                float4* dst = reinterpret_cast<float4*>(p.part + (2LL * c + (began ? 0 : 1)) * p.dim + col);
                dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
              }
            }
            first = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = 0.f;
          }
        }
      }
    }
  }
  if (ADD) return;
  const long long groups = (p.rows + ES_ZERO - 1) / ES_ZERO;
  const int vecs = p.dim / (F32 ? 4 : 8);
  for (long long g = warp; g < groups; g += stride) {
    const int row = (int)g * ES_ZERO + lane;
    unsigned none = __ballot_sync(0xffffffffu, lane < ES_ZERO && row < p.rows && p.range[row].y == 0);
    for (; none; none &= none - 1) {
      uint4* dst = static_cast<uint4*>(p.dtable) + (g * ES_ZERO + __ffs(none) - 1) * vecs;
      for (int i = lane; i < vecs; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
    }
  }
}

template <bool F32, bool ADD>
__global__ void __launch_bounds__(EJ_WARPS * 32)
embedding_join_kernel(const EmbGrad p) {
  if (!chain_begin()) return;
  __shared__ float s_part[EJ_WARPS][256];
  __shared__ long long s_long[EJ_WARPS];
  __shared__ int s_longs;
  const int warp = warp_index(), lane = threadIdx.x & 31, blocks = (p.dim + 255) / 256;
  const int valid = *p.valid;
  const long long items = (long long)(valid / p.chunk) * blocks;
  // the parts from .. to of an id that begins in chunk c (the first one is its second part, the others first parts)
  auto add_up = [&](int c, int col, int from, int to, float* acc) {
#pragma unroll 4
    for (int k = from; k <= to; ++k) {
      const float4* src = reinterpret_cast<const float4*>(p.part + (2LL * k + (k == c ? 1 : 0)) * p.dim + col);
      const float4 a = src[0], b = src[1];
      acc[0] += a.x; acc[1] += a.y; acc[2] += a.z; acc[3] += a.w;
      acc[4] += b.x; acc[5] += b.y; acc[6] += b.z; acc[7] += b.w;
    }
  };
  for (long long base = blockIdx.x; base < items; base += (long long)gridDim.x * EJ_WARPS) {
    if (threadIdx.x == 0) s_longs = 0;
    __syncthreads();
    const long long item = base + (long long)warp * gridDim.x;
    if (item < items) {
      const int c = (int)(item / blocks), col = (int)(item % blocks) * 256 + lane * 8, end = (c + 1) * p.chunk;
      const int row = p.sorted[end - 1];
      const int2 r = p.range[row];
      if (r.x >= c * p.chunk && r.x + r.y > end) {       // it begins in the chunk and goes on behind it
        const int last = (r.x + r.y - 1) / p.chunk;
        if (last - c < EJ_LONG) {
          if (col < p.dim) {
            float acc[8] = {};
            add_up(c, col, c, last, acc);
            emb_store<F32>(p.dtable, (long long)row * p.dim + col, acc, p.scale, ADD);
          }
        } else if (lane == 0) {
          s_long[atomicAdd(&s_longs, 1)] = item;       // (in any order: each is a result of its own)
        }
      }
    }
    __syncthreads();
    const int longs = s_longs;
    for (int i = 0; i < longs; ++i) {
      const int c = (int)(s_long[i] / blocks), col = (int)(s_long[i] % blocks) * 256 + lane * 8;
      const int row = p.sorted[(c + 1) * p.chunk - 1];
      const int2 r = p.range[row];
      const int n = (r.x + r.y - 1) / p.chunk - c + 1, from = c + (int)((long long)n * warp / EJ_WARPS);
      const int to = c + (int)((long long)n * (warp + 1) / EJ_WARPS) - 1;
      float acc[8] = {};
      if (col < p.dim) add_up(c, col, from, to, acc);
#pragma unroll
      for (int e = 0; e < 8; ++e) s_part[warp][lane * 8 + e] = acc[e];
      __syncthreads();
      if (warp == 0 && col < p.dim) {
        for (int w = 1; w < EJ_WARPS; ++w)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += s_part[w][lane * 8 + e];
        emb_store<F32>(p.dtable, (long long)row * p.dim + col, acc, p.scale, ADD);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// Tokens to a chunk: 32, more where the parts would take more than a few thousand rows.
static int emb_chunk(int tokens) {
  int c = 32;
  while (tokens / c > 4096) c *= 2;
  return c;
}
static int emb_per(int rows) {
  const int sms = sm_count(), even = (rows + sms - 1) / sms;
  return even < 64 ? 64 : even > EP_ROWS ? EP_ROWS : even;
}
static long long emb_align(long long n) { return (n + 15) / 16 * 16; }

struct EmbLayout {
  long long range, order, sorted, valid, part, bytes;
  EmbLayout(int tokens, int rows, int dim) {
    const int chunk = emb_chunk(tokens);
    const long long chunks = (tokens + chunk - 1) / chunk;
    range = 0;
    order = emb_align(range + 8LL * rows);
    sorted = emb_align(order + 4LL * tokens);
    valid = emb_align(sorted + 4LL * tokens);
    part = valid + 16;
    bytes = part + chunks * 2 * dim * 4;
  }
};

template <bool F32, bool ADD>
static void launch_embedding_grad(const EmbGrad& p, cudaStream_t stream) {
  const int sms = sm_count();
  chain(embedding_sum_kernel<F32, ADD>, 6 * sms, 256, 0, stream, p);
  if (p.tokens > p.chunk) chain(embedding_join_kernel<F32, ADD>, sms, EJ_WARPS * 32, 0, stream, p);
}

}  // namespace tpb

using namespace tpb;

// out[t] = scale * table[ids[t] - row0]; zeros for ids without a row here.
extern "C" int tpb_embedding_fwd(const void* table, const long long* ids, void* out, int tokens, int dim, long long vocab,
                                 long long row0, float scale, void* stream) {
  if (dim % 8 || dim <= 0 || reinterpret_cast<uintptr_t>(table) % 16 || reinterpret_cast<uintptr_t>(out) % 16) return -2;
  if (tokens <= 0) return 0;
  const unsigned nvec = dim / 8, blocks = (nvec + 127) / 128;
  const unsigned long long units = (unsigned long long)blocks * tokens;
  if (units > 0xffffffffu) return -2;
  const unsigned grid = (unsigned)((units + 7) / 8);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (scale == 1.f)
    chain(embedding_fwd_kernel<false>, grid, 256, 0, st, (const uint4*)table, ids, (uint4*)out, (unsigned)units, blocks, (int)nvec, vocab,
          row0, scale);
  else
    chain(embedding_fwd_kernel<true>, grid, 256, 0, st, (const uint4*)table, ids, (uint4*)out, (unsigned)units, blocks, (int)nvec, vocab,
          row0, scale);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

// Bytes of scratch for tpb_embedding_bwd.
extern "C" long long tpb_embedding_bwd_scratch(int tokens, int rows_local, int dim) {
  return EmbLayout(tokens, rows_local, dim).bytes;
}

// dtable[v] = (`add`: dtable[v] +) scale * sum of dout[t] over ids[t] = row0 + v; with `add`, rows without a token are left alone.
extern "C" int tpb_embedding_bwd(const void* dout, const long long* ids, void* dtable, void* scratch, int tokens, int dim, int rows_local,
                                 long long row0, int dtable_is_f32, int add, float scale, void* stream) {
  if (dim % 8 || dim <= 0 || tokens < 0 || rows_local < 0) return -2;
  for (const void* a : {dout, (const void*)dtable, (const void*)scratch})
    if (reinterpret_cast<uintptr_t>(a) % 16) return -2;
  if (rows_local == 0 || (tokens == 0 && add)) return 0;
  const EmbLayout at(tokens, rows_local, dim);
  char* s = static_cast<char*>(scratch);
  EmbGrad p = {};
  p.ids = ids;
  p.dout = static_cast<const __nv_bfloat16*>(dout);
  p.dtable = dtable;
  p.range = reinterpret_cast<int2*>(s + at.range);
  p.order = reinterpret_cast<int*>(s + at.order);
  p.sorted = reinterpret_cast<int*>(s + at.sorted);
  p.valid = reinterpret_cast<int*>(s + at.valid);
  p.part = reinterpret_cast<float*>(s + at.part);
  p.row0 = row0;
  p.tokens = tokens;
  p.rows = rows_local;
  p.dim = dim;
  p.chunk = emb_chunk(tokens);
  p.chunks = (tokens + p.chunk - 1) / p.chunk;
  p.per = emb_per(rows_local);
  p.scale = scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int smem = EP_WARPS * p.per * 4;
  static std::atomic<unsigned> ready{0};              // a bit for each device
  int device = 0;
  cudaError_t set = cudaGetDevice(&device);
  if (set == cudaSuccess && (device > 31 || !(ready.load(std::memory_order_relaxed) >> device & 1))) {
    set = cudaFuncSetAttribute(embedding_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EP_WARPS * EP_ROWS * 4);
    if (set == cudaSuccess && device <= 31) ready.fetch_or(1u << device, std::memory_order_relaxed);
  }
  if (set != cudaSuccess) return 1000 + (int)set;
  chain(embedding_plan_kernel, (rows_local + p.per - 1) / p.per, EP_WARPS * 32, smem, st, p);
  if (dtable_is_f32) add ? launch_embedding_grad<true, true>(p, st) : launch_embedding_grad<true, false>(p, st);
  else add ? launch_embedding_grad<false, true>(p, st) : launch_embedding_grad<false, false>(p, st);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
