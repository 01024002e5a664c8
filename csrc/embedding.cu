// Embedding: rows of a table, scaled, and the table's gradient by sorted tokens.
//
//   out[t] = scale * E[id[t]],   dE[v] (+)= scale * sum of dout[t] over the tokens t with id[t] = v.
//
// Both are bound by memory.  The gradient of a training step writes the whole table (most rows as zeros) and reads dout once;
// what makes it slow otherwise are atomics, which read and write an fp32 table that has to be zeroed before and rounded behind, in an
// order that differs from run to run.  Here every row has one writer, and the order of its sum follows from the ids alone: a chunk's tokens
// ascending, then the chunks' parts ascending or, of an id with many, in 32 shares of them:
//
// * embedding_plan_kernel puts the tokens in order of their ids.  A CTA has a set of ids (every sets-th one, so that frequent ones, which
//   have low numbers, are spread) and looks at all tokens, so no CTA has to wait for another: its 32 warps count what each id has in their
//   parts of the tokens, the counts become places (how many tokens the sets in front have is counted on the way), and a second
//   look puts the tokens there, in order.  Up to 8192 tokens a warp keeps its part in registers between the looks (9 us); more
//   are turned into codes by a kernel of their own first, and the second look is at a list of the set's (65536 tokens, 0.3 of them of
//   one id: 45 us -> 3 + 20).
// * embedding_sum_kernel cuts that order into chunks of equal size, whatever the ids: a warp adds up 256 columns of a chunk's rows
//   in fp32.  An id whose tokens lie within a chunk is written at once; one that reaches over a chunk's border leaves its part, at most
//   two a chunk.  Then some warps write zeros to the rows without a token, handed out by a counter: in equal shares they waited for
//   the warps whose chunks took long (204 -> 192 us); all warps' writes at once are slower than a quarter's.
// * embedding_join_kernel adds up the parts in the chunks' order, an id to a warp, or one with many (the padding's row) to a CTA.  (Joined by
//   whoever leaves the last part, with fences and counters, it all took longer: 65536 tokens 134 -> 148 us.)
//
// Few tokens take two other kernels, embedding_rank_kernel and embedding_run_kernel, which have no more to do than the tokens ask for.  (Added up by
// atomics in L2, red.v4.f32, the rows of the many tokens' form took longer, too: 8192 of 128256 x 4096 67 -> 86 us.)
//
// 8192 tokens of a 128256 x 4096 table: 170 us for 1.12 GB, 171 at a copy's rate; 65536 of 32000 x 2048, 0.3 of them of one id: 103 us for 0.4 GB.

#include <atomic>

#include "common.cuh"
#include "tpb.h"

namespace tpb {

int sm_count();

constexpr int EP_WARPS = 32;                 // of the planning kernel
constexpr int EP_ROWS = 1024;                // most ids to a CTA of it
constexpr int EP_BATCH = 8;                  // ids of a lane that are asked for at once
constexpr int EP_SMEM = 220 * 1024;
constexpr int EJ_WARPS = 32;                 // of the joining kernel
// Chunks behind its first from which a CTA's warps share an id.  8192 tokens, and 65536 with 0.3 of one id (when all took 177 and 127 us): 4 177.0
// and 126.7, 8 176.8 and 126.6, 16 178.6 and 126.8.
constexpr int EJ_LONG = 8;
// Of the summing kernel: CTAs to an SM, rows that a warp asks for ahead, and warps of a CTA that write zeros at the end.  us, 8192 tokens of a 128256 x
// 4096 table / 65536 of 32000 x 2048, 0.3 of them of one id: 4, 8, 2 170 / 103;  4, 8, 4 175 / 103;  4, 8, 8 184 / 103;  3, 16, 8 180 / 111;  2, 16, 8
// 198 / 125;  5, 8, 8 - / 129;  two CTAs with eight rows in registers, 8 177 / 127.
constexpr int ES_CTAS = 4, ES_AHEAD = 8, ES_FILL = 2;
constexpr int ES_ZERO = 4;                   // rows that a warp of it looks at for ones without tokens

__device__ __forceinline__ void emb_unpack(const uint4& u, float* f) {
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
}
__device__ __forceinline__ uint4 emb_pack(const float* f) {
  return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}

// A warp takes up to 4 x 32 vectors of a token's row, all asked for before the first is used.  4099 rows of 5120 11.6 us, 12.8 at a copy's rate (some
// rows come from L2 a second time).
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

// Scratch of the gradient, in this order: range [rows] (first place, tokens), order [tokens] (the last one of an id is marked), number of
// tokens that have a row, a counter, codes [tokens, padded], parts.
struct EmbGrad {
  const long long* ids;
  const __nv_bfloat16* dout;
  void* dtable;
  int2* range;
  unsigned *order, *codes;
  int *valid, *taken;                        // taken (zeroed by the planning kernel): rows that the sum's warps have looked at
  float* part;                               // [chunks][2][dim]: of the id that began before the chunk, of the one that goes on behind it
  long long row0;
  int tokens, rows, dim, chunk;
  int sets, per, share;                      // CTAs of the planning kernel, most ids to one: id v is the v / sets-th of set v % sets; tokens to a warp
  int list;                                  // entries of a warp's list there
  unsigned inv, shift;                       // v / sets = v * inv >> shift
  float scale;
};

constexpr unsigned EMB_LAST = 1u << 31, EMB_NONE = ~0u;

// An id as its set and its number there; EMB_NONE: it has no row.
__device__ __forceinline__ unsigned emb_code(const EmbGrad& p, long long id) {
  const unsigned v = (unsigned)id, q = (unsigned)((unsigned long long)v * p.inv >> p.shift);
  return id < 0 || id >= p.rows ? EMB_NONE : (v - q * p.sets) * EP_ROWS + q;
}

// Codes of all tokens: where there are many, the planning kernel's CTAs do not all work them out.
__global__ void __launch_bounds__(256)
embedding_code_kernel(const EmbGrad p) {
  if (!chain_begin()) return;
  const int t = blockIdx.x * 256 + threadIdx.x, all = EP_WARPS * p.share;
  if (t < all) p.codes[t] = t < p.tokens ? emb_code(p, p.ids[t] - p.row0) : EMB_NONE;
}

// CODES: the tokens' codes come from the kernel before, and a warp lists those of its part that are the CTA's (if the list is too short
// for them it looks at all of them again).  Else a warp has EP_BATCH tokens a lane at most and keeps them.
template <bool CODES>
__global__ void __launch_bounds__(EP_WARPS * 32)
embedding_plan_kernel(const EmbGrad p) {
  if (!chain_begin()) return;
  extern __shared__ __align__(16) int ep_hist[];           // [warps][per], ends [per], lists [warps][list]; per a multiple of 4
  __shared__ int s_warp[EP_WARPS], s_below;
  const int warp = warp_index(), lane = threadIdx.x & 31, set = blockIdx.x;
  const unsigned least = set * EP_ROWS, below_me = (1u << lane) - 1;
  const int t0 = warp * p.share;             // (the codes are padded; a launch without has at most 2^13 tokens)
  int* hist = ep_hist + warp * p.per;
  int* ends = ep_hist + EP_WARPS * p.per;
  unsigned* list = reinterpret_cast<unsigned*>(ends + p.per) + warp * p.list;
  unsigned code[EP_BATCH];
  if (!CODES) {
    long long id[EP_BATCH];
#pragma unroll
    for (int i = 0; i < EP_BATCH; ++i) {
      const int t = t0 + 32 * i + lane;
      id[i] = 32 * i < p.share && t < p.tokens ? p.ids[t] - p.row0 : -1;
    }
#pragma unroll
    for (int i = 0; i < EP_BATCH; ++i) code[i] = emb_code(p, id[i]);
  }
  for (int i = threadIdx.x; i < EP_WARPS * p.per / 4; i += EP_WARPS * 32) reinterpret_cast<int4*>(ep_hist)[i] = make_int4(0, 0, 0, 0);
  if (threadIdx.x == 0) {
    s_below = 0;
    if (set == 0) *p.taken = 0;
  }
  __syncthreads();
  // ---- which tokens of the warp's part have an id of this set, and how many one of a set in front
  int below = 0, hits = 0;
  if (CODES) {
    for (int t = 0; t < p.share; t += 256) {
      unsigned c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = p.codes[t0 + t + 32 * i + lane];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = c[i] - least < EP_ROWS;
        const unsigned who = __ballot_sync(0xffffffffu, in);
        below += c[i] < least;
        if (who == 0) continue;
        const int at = hits + __popc(who & below_me);
        if (in && at < p.list) list[at] = (unsigned)(t + 32 * i + lane) * EP_ROWS | (c[i] - least);
        hits += __popc(who);
      }
    }
    __syncwarp();
  } else {
#pragma unroll
    for (int i = 0; i < EP_BATCH; ++i) below += code[i] < least;
  }
  // f(has, number of the id, token) for the warp's tokens, 32 at a time and in order; those of the set are enough
  auto each = [&](auto&& f) {
    if (!CODES) {
#pragma unroll
      for (int i = 0; i < EP_BATCH; ++i)
        if (__any_sync(0xffffffffu, code[i] - least < EP_ROWS)) f(code[i] - least < EP_ROWS, code[i] - least, t0 + 32 * i + lane);
    } else if (hits <= p.list) {
      for (int i = 0; i < hits; i += 32) {
        const unsigned e = i + lane < hits ? list[i + lane] : 0;
        f(i + lane < hits, e % EP_ROWS, t0 + (int)(e / EP_ROWS));
      }
    } else {
#pragma unroll 4
      for (int t = 0; t < p.share; t += 32) {
        const unsigned v = p.codes[t0 + t + lane] - least;
        f(v < EP_ROWS, v, t0 + t + lane);
      }
    }
  };
  // ---- how many each id has in each warp's part; many may have one and the same (the padding's)
  each([&](bool has, unsigned r, int) {
    const unsigned who = __ballot_sync(0xffffffffu, has);
    if (who == 0) return;
    const int leader = __ffs(who) - 1;
    const unsigned first = __shfl_sync(0xffffffffu, r, leader), same = __ballot_sync(0xffffffffu, has && r == first);
    if (lane == leader) atomicAdd(&hist[r], __popc(same));
    else if (has && !(same >> lane & 1)) atomicAdd(&hist[r], 1);
  });
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0 && below) atomicAdd(&s_below, below);
  __syncthreads();
  // ---- their places: a thread for each id
  const int r = threadIdx.x, row = r * p.sets + set;
  const bool has_row = r < p.per && row < p.rows;
  int before[EP_WARPS], count = 0;
#pragma unroll
  for (int w = 0; w < EP_WARPS; ++w) before[w] = has_row ? ep_hist[w * p.per + r] : 0;
#pragma unroll
  for (int w = 0; w < EP_WARPS; ++w) {
    const int n = before[w];
    before[w] = count;
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
  const int start = s_below + sum - count + __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[lane] : 0);
  if (has_row) {
#pragma unroll
    for (int w = 0; w < EP_WARPS; ++w) ep_hist[w * p.per + r] = start + before[w];
    ends[r] = start + count - 1;
    p.range[row] = make_int2(start, count);
  }
  if (set == p.sets - 1 && r == EP_WARPS * 32 - 1) *p.valid = start + count;
  __syncthreads();
  // ---- the tokens, in order: those of one id in a warp's 32 by lane
  each([&](bool has, unsigned r, int t) {
    const unsigned any = __ballot_sync(0xffffffffu, has);
    if (has) {
      const unsigned same = __match_any_sync(any, r), lower = same & below_me;
      const int at = hist[r] + __popc(lower);
      p.order[at] = t | (at == ends[r] ? EMB_LAST : 0);
      __syncwarp(any);
      if (lower == 0) hist[r] = at + __popc(same);
    }
    __syncwarp();
  });
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

// One column of a row.
template <bool F32>
__device__ __forceinline__ void emb_store1(void* dtable, long long at, float a, float scale, bool add) {
  a = mul_exact(a, scale);
  if (F32) {
    float* dst = static_cast<float*>(dtable) + at;
    *dst = add ? *dst + a : a;
  } else {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(dtable) + at;
    *dst = __float2bfloat16(add ? __bfloat162float(*dst) + a : a);
  }
}

// Sixteen bytes to this thread's own place in shared memory.
__device__ __forceinline__ void emb_ask(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

template <bool F32, bool ADD>
__global__ void __launch_bounds__(256, ES_CTAS)
embedding_sum_kernel(const EmbGrad p) {
  if (!chain_begin()) return;
  __shared__ uint4 mem[ES_AHEAD][256];       // a thread's own columns of the rows that are under way
  const int lane = threadIdx.x & 31, blocks = (p.dim + 255) / 256;
  const int valid = *p.valid, warps = gridDim.x * 8;
  const int items = (valid + p.chunk - 1) / p.chunk * blocks;
  for (int item = blockIdx.x * 8 + warp_index(); item < items; item += warps) {
    const int c = item / blocks, col = (item - c * blocks) * 256 + lane * 8, base = c * p.chunk;
    const int n = min(p.chunk, valid - base);
    const bool has = col < p.dim;
    float acc[8] = {};
    unsigned here = lane < n ? p.order[base + lane] : EMB_LAST;
    bool began = base > 0 && !(p.order[base - 1] & EMB_LAST);        // the first id began before the chunk
    const __nv_bfloat16* from = p.dout + (has ? col : 0);
    auto fetch = [&](unsigned tokens, int j, bool there) {             // row j of 32; a group each time
      const int t = __shfl_sync(0xffffffffu, tokens, j & 31) & ~EMB_LAST;
      if (there && has) emb_ask(&mem[j % ES_AHEAD][threadIdx.x], from + (long long)t * p.dim);        // (what is asked for is also waited for)
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int j = 0; j < ES_AHEAD; ++j) fetch(here, j, j < n);
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int m = min(32, n - i0), left = n - i0 - 32;
      const unsigned next = lane < left ? p.order[base + i0 + 32 + lane] : EMB_LAST;
      const unsigned last = __ballot_sync(0xffffffffu, here & EMB_LAST), ends = last | (i0 + m == n ? 1u << (m - 1) : 0);
      const int row = ends >> lane & 1 && lane < m ? (int)(p.ids[here & ~EMB_LAST] - p.row0) : 0;
#pragma unroll 4
      for (int j = 0; j < m; ++j) {
        asm volatile("cp.async.wait_group %0;" ::"n"(ES_AHEAD - 1) : "memory");
        float x[8];
        emb_unpack(mem[j % ES_AHEAD][threadIdx.x], x);
        const int k = j + ES_AHEAD;
        fetch(k < 32 ? here : next, k, i0 + k < n);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += x[e];
        if (ends >> j & 1) {
          const int id = __shfl_sync(0xffffffffu, row, j);
          if (has) {
            if (began || !(last >> j & 1)) {
              float4* dst = reinterpret_cast<float4*>(p.part + (2LL * c + (began ? 0 : 1)) * p.dim + col);
              dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
              dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
            } else {
              emb_store<F32>(p.dtable, (long long)id * p.dim + col, acc, p.scale, ADD);
            }
          }
          began = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        }
      }
      here = next;
    }
  }
  if (ADD || warp_index() >= ES_FILL) return;
  // rows without a token, to whoever is free (warps end their chunks at times that differ by a fourth of the kernel's)
  const int groups = (p.rows + ES_ZERO - 1) / ES_ZERO, vecs = p.dim / (F32 ? 4 : 8);
  auto take = [&]() { return lane == 0 ? atomicAdd(p.taken, 1) : 0; };
  for (int ahead = take();;) {
    const int group = __shfl_sync(0xffffffffu, ahead, 0), row = group * ES_ZERO + lane;
    if (group >= groups) break;
    ahead = take();
    unsigned none = __ballot_sync(0xffffffffu, lane < ES_ZERO && row < p.rows && p.range[row].y == 0);
    for (; none; none &= none - 1) {
      uint4* dst = static_cast<uint4*>(p.dtable) + ((long long)group * ES_ZERO + __ffs(none) - 1) * vecs;
      for (int i = lane; i < vecs; i += 32) dst[i] = make_uint4(0, 0, 0, 0);
    }
  }
}

template <bool F32, bool ADD>
__global__ void __launch_bounds__(EJ_WARPS * 32)
embedding_join_kernel(const EmbGrad p) {
  if (!chain_begin()) return;
  __shared__ __align__(16) float s_part[EJ_WARPS][256];
  __shared__ int4 s_long[EJ_WARPS];          // id, first and last chunk, columns
  __shared__ int s_longs;
  const int warp = warp_index(), lane = threadIdx.x & 31, blocks = (p.dim + 255) / 256;
  const int items = *p.valid / p.chunk * blocks;
  // the parts from .. to of an id that begins in chunk c (that one's is its second, the others' are first ones)
  auto add_up = [&](int c, int col, int from, int to, float* acc) {
#pragma unroll 4
    for (int k = from; k <= to; ++k) {
      const float4* src = reinterpret_cast<const float4*>(p.part + (2LL * k + (k == c ? 1 : 0)) * p.dim + col);
      const float4 a = src[0], b = src[1];
      acc[0] += a.x; acc[1] += a.y; acc[2] += a.z; acc[3] += a.w;
      acc[4] += b.x; acc[5] += b.y; acc[6] += b.z; acc[7] += b.w;
    }
  };
  for (int base = blockIdx.x; base < items; base += gridDim.x * EJ_WARPS) {
    if (threadIdx.x == 0) s_longs = 0;
    __syncthreads();
    const int item = base + warp * gridDim.x;
    if (item < items) {
      const int c = item / blocks, col0 = (item - c * blocks) * 256, col = col0 + lane * 8;
      const unsigned end = p.order[(c + 1) * p.chunk - 1];
      if (!(end & EMB_LAST)) {               // an id goes on behind the chunk
        const int row = (int)(p.ids[end] - p.row0);
        const int2 r = p.range[row];
        const int last = (r.x + r.y - 1) / p.chunk;
        if (r.x < c * p.chunk) {             // and began before it: whoever has that chunk looks after it
        } else if (last - c < EJ_LONG) {
          if (col < p.dim) {
            float acc[8] = {};
            add_up(c, col, c, last, acc);
            emb_store<F32>(p.dtable, (long long)row * p.dim + col, acc, p.scale, ADD);
          }
        } else if (lane == 0) {
          s_long[atomicAdd(&s_longs, 1)] = make_int4(row, c, last, col0);       // (in any order: each is a result of its own)
        }
      }
    }
    __syncthreads();
    const int longs = s_longs;
    for (int i = 0; i < longs; ++i) {
      const int4 it = s_long[i];
      const int n = it.z - it.y + 1, from = it.y + (int)((long long)n * warp / EJ_WARPS);
      const int to = it.y + (int)((long long)n * (warp + 1) / EJ_WARPS) - 1;
      float acc[8] = {};
      if (it.w + lane * 8 < p.dim) add_up(it.y, it.w + lane * 8, from, to, acc);
      reinterpret_cast<float4*>(s_part[warp])[2 * lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      reinterpret_cast<float4*>(s_part[warp])[2 * lane + 1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      __syncthreads();
      const int col = it.w + threadIdx.x;
      if (threadIdx.x < 256 && col < p.dim) {
        float a = s_part[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < EJ_WARPS; ++w) a += s_part[w][threadIdx.x];
        emb_store1<F32>(p.dtable, (long long)it.x * p.dim + col, a, p.scale, ADD);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// ---- few tokens: each is compared with all the others, once, and then every id's run of the order has a warp to itself.  Nothing is counted
// for ids without a token, and no parts are joined.  Gradients that are added, up to EF_MOST tokens; us, this / the three kernels above, ids evenly
// spread and half of them one, fp32: 64 tokens of 128256 x 4096 4.9 / 25.5 and 4.9 / 19.5, 1024 11 / 28 and 10.5 / 28, 4096 37 / 50 and 36 / 49; 4096 of
// 2000 x 1024 14 / 16 and 21 / 19 (8192, when a long run still took longer: 28 / 18).  Gradients that are written, for which the ranking
// kernel zeroes the table as well, up to EF_WRITTEN, bf16: 64 of 128256 x 4096 145 / 153, 2048 of 32000 x 2048 27 / 31 and 29 / 32, of 2000 x 1024
// 10.6 / 13.3 and 12.6 / 14.6; 4096 of them 14.2 / 14.2 and 21 / 17.
constexpr int EF_MOST = 4096, EF_WRITTEN = 2048;
constexpr int EF_WARPS = 16;                 // of the ranking kernel
constexpr int EF_ZEROS = 16;                 // vectors of a thread of it that writes zeros

struct EmbFew {
  const long long* ids;
  const __nv_bfloat16* dout;
  void* dtable;
  int2* order;                               // [tokens]: a token and its row, or -1 (those are last); by row, then by token
  long long row0;
  int tokens, rows, dim;
  int rankers;                               // CTAs that rank
  int longs, blocks;                         // CTAs to a team for long runs; blocks of ER_VECS x 256 columns
  long long zeros;                           // vectors of the table, if it is written
  float scale;
};

// The place of a token is how many stand in front: those of lower rows, and of its own row those with lower numbers.  A warp compares its token with
// all of them, which the CTA has as rows in shared memory: two instructions each.  The CTAs behind write zeros to the table.
__global__ void __launch_bounds__(EF_WARPS * 32)
embedding_rank_kernel(const EmbFew p) {
  if (!chain_begin()) return;
  if ((int)blockIdx.x >= p.rankers) {
    uint4* dst = static_cast<uint4*>(p.dtable);
    const long long i0 = (blockIdx.x - p.rankers) * (EF_WARPS * 32LL * EF_ZEROS) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < EF_ZEROS; ++i)
      if (i0 + EF_WARPS * 32 * i < p.zeros) dst[i0 + EF_WARPS * 32 * i] = make_uint4(0, 0, 0, 0);
    return;
  }
  __shared__ __align__(16) unsigned s_row[EF_MOST];
  const int lane = threadIdx.x & 31, t = blockIdx.x * EF_WARPS + warp_index(), all = (p.tokens + 3) / 4 * 4;      // (up to EF_MOST)
#pragma unroll 4
  for (int i = threadIdx.x; i < all; i += EF_WARPS * 32) {
    const long long id = i < p.tokens ? p.ids[i] - p.row0 : -1;
    s_row[i] = id < 0 || id >= p.rows ? EMB_NONE : (unsigned)id;
  }
  __syncthreads();
  if (t >= p.tokens) return;
  const unsigned me = s_row[t];
  int less = 0, i = lane * 4;
#pragma unroll 4
  for (; i + 4 <= t; i += 128) {
    const uint4 c = *reinterpret_cast<const uint4*>(s_row + i);
    less += (c.x <= me) + (c.y <= me) + (c.z <= me) + (c.w <= me);
  }
  if (i <= t) {                              // the vector that it is in
    for (int k = i; k < i + 4; ++k) less += k < t ? s_row[k] <= me : s_row[k] < me;
    i += 128;
  }
#pragma unroll 4
  for (; i < all; i += 128) {
    const uint4 c = *reinterpret_cast<const uint4*>(s_row + i);
    less += (c.x < me) + (c.y < me) + (c.z < me) + (c.w < me);
  }
  less = __reduce_add_sync(0xffffffffu, less);
  if (lane == 0) p.order[less] = make_int2(t, (int)me);      // (EMB_NONE: -1)
}

// Old numbers of eight columns, loaded ahead of their sum.
template <bool F32>
struct EmbOld {
  uint4 a, b;
  __device__ __forceinline__ void load(const void* dtable, long long at) {
    if (F32) {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(dtable) + at);
      a = src[0];
      b = src[1];
    } else {
      a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(dtable) + at);
    }
  }
  __device__ __forceinline__ void add_to(float* f) const {
    float o[8];
    if (F32) {
      o[0] = __uint_as_float(a.x); o[1] = __uint_as_float(a.y); o[2] = __uint_as_float(a.z); o[3] = __uint_as_float(a.w);
      o[4] = __uint_as_float(b.x); o[5] = __uint_as_float(b.y); o[6] = __uint_as_float(b.z); o[7] = __uint_as_float(b.w);
    } else {
      emb_unpack(a, o);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += o[e];
  }
};
template <bool F32>
__device__ __forceinline__ void emb_write(void* dtable, long long at, const float* f) {
  if (F32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(dtable) + at);
    dst[0] = make_float4(f[0], f[1], f[2], f[3]);
    dst[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(dtable) + at) = emb_pack(f);
  }
}

// Runs of the order, a warp to each of less than ER_LONG tokens and ER_VECS x 256 columns, in ascending order: the old numbers and the first row are
// asked for at once, then eight rows at a time.
// Longer ones: the first p.longs x ER_TEAMS CTAs, 64 columns each.  A team looks through the order for the runs that are its own (by their place, at
// most one in ER_LONG); a warp takes one, a fourth of its lanes every fourth row, or, from ER_ALL tokens on, the whole CTA.  2048 tokens of 128256 x 4096,
// fp32, 16 us (13 at a copy's rate for what is read and written), behind 6 of ranking: it ends soon after it has got going.  us: a CTA of 16 warps for
// 16 places and 256 columns, with barriers for the long runs, 38 for both kernels, now 21; two rows at a time instead of eight 20 to 24 with frequent ids.
constexpr int ER_WARPS = 8, ER_VECS = 2, ER_TEAMS = 4, ER_LONG = 32, ER_ALL = 128;

// Rows j0, j0 + step, ... by 32, of the run of `row` that begins at `from`, added up for a lane's eight columns, then over the warp's fourths.
__device__ __forceinline__ void emb_run(const EmbFew& p, int from, int row, int j0, int step, int col, float* acc) {
  const int lane = threadIdx.x & 31;
  const __nv_bfloat16* src = p.dout + (col < p.dim ? col : 0);
  auto tokens = [&](int j) {                 // of places j + lane of the run; -1 behind it
    const int at = from + j + lane;
    const int2 e = at < p.tokens ? p.order[at] : make_int2(0, -1);
    return e.y == row ? e.x : -1;
  };
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  int here = tokens(j0);
  while (__shfl_sync(0xffffffffu, here, 0) >= 0) {
    uint4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = __shfl_sync(0xffffffffu, here, 4 * i + lane / 8);
      v[i] = t >= 0 && col < p.dim ? *reinterpret_cast<const uint4*>(src + (long long)t * p.dim) : make_uint4(0, 0, 0, 0);
    }
    j0 += step;
    here = tokens(j0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x[8];
      emb_unpack(v[i], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += x[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 8);
    acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 16);
  }
}

template <bool F32, bool ADD>
__global__ void __launch_bounds__(ER_WARPS * 32, 4)
embedding_run_kernel(const EmbFew p) {
  if (!chain_begin()) return;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  auto row_at = [&](int i) { return i >= 0 && i < p.tokens ? p.order[i].y : -1; };
  if (blockIdx.x < (unsigned)p.longs * ER_TEAMS) {
    __shared__ int s_run[EF_MOST / ER_LONG], s_all[EF_MOST / ER_ALL], s_runs, s_alls;
    __shared__ __align__(16) float s_part[ER_WARPS][64];
    const int team = blockIdx.x % ER_TEAMS, col0 = blockIdx.x / ER_TEAMS * 64, col = col0 + lane % 8 * 8;
    if (threadIdx.x == 0) s_runs = s_alls = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = threadIdx.x; i < p.tokens; i += ER_WARPS * 32) {
      const int row = row_at(i);
      if (row < 0 || row_at(i + ER_LONG - 1) != row || row_at(i - 1) == row || i / ER_LONG % ER_TEAMS != team) continue;
      if (row_at(i + ER_ALL - 1) == row) s_all[atomicAdd(&s_alls, 1)] = i;        // (in any order: each is a result of its own)
      else s_run[atomicAdd(&s_runs, 1)] = i;
    }
    __syncthreads();
    const int runs = s_runs, alls = s_alls;
    float acc[8];
    for (int k = 0; k < alls; ++k) {
      const int row = row_at(s_all[k]);
      emb_run(p, s_all[k], row, warp * 32, ER_WARPS * 32, col, acc);
      if (lane < 8) {
        reinterpret_cast<float4*>(s_part[warp])[2 * lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        reinterpret_cast<float4*>(s_part[warp])[2 * lane + 1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      }
      __syncthreads();
      if (threadIdx.x < 64 && col0 + (int)threadIdx.x < p.dim) {
        float a = s_part[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < ER_WARPS; ++w) a += s_part[w][threadIdx.x];
        emb_store1<F32>(p.dtable, (long long)row * p.dim + col0 + threadIdx.x, a, p.scale, ADD);
      }
      __syncthreads();
    }
    for (int k = warp; k < runs; k += ER_WARPS) {
      const int row = row_at(s_run[k]);
      emb_run(p, s_run[k], row, 0, 32, col, acc);
      if (lane < 8 && col < p.dim) emb_store<F32>(p.dtable, (long long)row * p.dim + col, acc, p.scale, ADD);
    }
    return;
  }
  const unsigned unit = (blockIdx.x - p.longs * ER_TEAMS) * ER_WARPS + warp;
  const int at = unit / p.blocks, col = (unit - at * p.blocks) * (ER_VECS * 256) + lane * 8;
  if (at >= p.tokens) return;
  const int2 here = at + lane < p.tokens ? p.order[at + lane] : make_int2(0, -1);
  const int row = __shfl_sync(0xffffffffu, here.y, 0), n = __ffs(__ballot_sync(0xffffffffu, here.y != row)) - 1;
  if (row < 0 || n < 0 || row_at(at - 1) == row) return;       // (no difference: ER_LONG or more)
  const long long to = (long long)row * p.dim + col;
  auto load = [&](int j, int i) {
    const int t = __shfl_sync(0xffffffffu, here.x, j & 31);
    return j < n && col + 256 * i < p.dim ? *reinterpret_cast<const uint4*>(p.dout + (long long)t * p.dim + col + 256 * i) : make_uint4(0, 0, 0, 0);
  };
  EmbOld<F32> old[ER_VECS];
  uint4 first[ER_VECS];
#pragma unroll
  for (int i = 0; i < ER_VECS; ++i) {
    first[i] = load(0, i);
    if (ADD && col + 256 * i < p.dim) old[i].load(p.dtable, to + 256 * i);
  }
#pragma unroll
  for (int i = 0; i < ER_VECS; ++i) {
    float acc[8];
    emb_unpack(first[i], acc);
    for (int j = 1; j < n; j += 8) {
      uint4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = load(j + k, i);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float x[8];
        emb_unpack(v[k], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += x[e];
      }
    }
    if (col + 256 * i < p.dim) {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = mul_exact(acc[e], p.scale);
      if (ADD) old[i].add_to(acc);
      emb_write<F32>(p.dtable, to + 256 * i, acc);
    }
  }
}

// Tokens to a chunk, by the items (a chunk's 256 columns) that chunks of 32 would make: 16 where those are few, so that more warps share the rows,
// 64 where they are many, for fewer parts to join; more where the parts would take thousands of rows.  us: 333 tokens of 1024 columns 12.1 with
// 16, 14.1 with 32; 16384 of 512 26.4, 29.0; 4099 of 2048 73.8, 73.7; 8192 of 4096 176, 170; 65536 of 2048 117 with 32, 102 with 64.
static int emb_chunk(int tokens, int dim) {
  const long long items = (tokens + 31LL) / 32 * ((dim + 255) / 256);
  int c = items < 2048 ? 16 : items < 8192 ? 32 : 64;
  while (tokens / c > 4096) c *= 2;
  return c;
}
static int emb_per(int rows) {
  const int sms = sm_count(), even = (rows + sms - 1) / sms;
  return even < 64 ? 64 : even > EP_ROWS ? EP_ROWS : (even + 3) / 4 * 4;
}
static long long emb_align(long long n) { return (n + 15) / 16 * 16; }

// Tokens to a warp of the planning kernel: whole rounds of it.
static int emb_share(int tokens) {
  const int round = tokens <= EP_WARPS * 32 * EP_BATCH ? 32 : 256;
  return (int)((tokens + (long long)EP_WARPS * round - 1) / (EP_WARPS * round)) * round;
}

struct EmbLayout {
  long long range, order, valid, codes, part, bytes;
  int chunk, chunks, share;
  bool coded;
  EmbLayout(int tokens, int rows, int dim) {
    chunk = emb_chunk(tokens, dim);
    chunks = (int)((tokens + (long long)chunk - 1) / chunk);
    share = emb_share(tokens);
    coded = tokens > EP_WARPS * 32 * EP_BATCH;
    range = 0;
    order = emb_align(range + 8LL * rows);
    valid = emb_align(order + 4LL * tokens);
    codes = valid + 16;
    part = codes + (coded ? 4LL * share * EP_WARPS : 0);
    bytes = part + 2LL * chunks * dim * 4;
  }
};

static bool emb_few(int tokens, int dim, bool add) { return tokens <= (add ? EF_MOST : EF_WRITTEN) && dim <= 1 << 20; }

template <bool F32, bool ADD>
static void launch_embedding_few(EmbFew& p, cudaStream_t stream) {
  constexpr long long PER = EF_WARPS * 32LL * EF_ZEROS;
  p.rankers = (p.tokens + EF_WARPS - 1) / EF_WARPS;
  p.zeros = ADD ? 0 : (long long)p.rows * p.dim / (F32 ? 4 : 8);
  chain(embedding_rank_kernel, (unsigned)(p.rankers + (p.zeros + PER - 1) / PER), EF_WARPS * 32, 0, stream, p);
  p.longs = p.tokens >= ER_LONG ? (p.dim + 63) / 64 : 0;
  p.blocks = (p.dim + ER_VECS * 256 - 1) / (ER_VECS * 256);
  if (p.tokens > 0)
    chain(embedding_run_kernel<F32, ADD>, p.longs * ER_TEAMS + (unsigned)(((long long)p.tokens * p.blocks + ER_WARPS - 1) / ER_WARPS), ER_WARPS * 32, 0,
          stream, p);
}

template <bool F32, bool ADD>
static void launch_embedding_grad(const EmbGrad& p, cudaStream_t stream) {
  const int sms = sm_count();
  chain(embedding_sum_kernel<F32, ADD>, ES_CTAS * sms, 256, 0, stream, p);
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
  const long long order = 8LL * tokens;      // of few tokens
  const long long all = emb_few(tokens, dim, false) ? 0 : EmbLayout(tokens, rows_local, dim).bytes;
  return all > order ? all : order;
}

// dtable[v] = (`add`: dtable[v] +) scale * sum of dout[t] over ids[t] = row0 + v; with `add`, rows without a token are left alone.
extern "C" int tpb_embedding_bwd(const void* dout, const long long* ids, void* dtable, void* scratch, int tokens, int dim, int rows_local,
                                 long long row0, int dtable_is_f32, int add, float scale, void* stream) {
  if (dim % 8 || dim <= 0 || tokens < 0 || tokens > 1 << 30 || rows_local < 0 || rows_local > 1 << 30) return -2;
  for (const void* a : {dout, (const void*)dtable, (const void*)scratch})
    if (reinterpret_cast<uintptr_t>(a) % 16) return -2;
  if (rows_local == 0 || (tokens == 0 && add)) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (emb_few(tokens, dim, add != 0)) {
    EmbFew p = {};
    p.ids = ids;
    p.dout = static_cast<const __nv_bfloat16*>(dout);
    p.dtable = dtable;
    p.order = static_cast<int2*>(scratch);
    p.row0 = row0;
    p.tokens = tokens;
    p.rows = rows_local;
    p.dim = dim;
    p.scale = scale;
    if (dtable_is_f32) add ? launch_embedding_few<true, true>(p, st) : launch_embedding_few<true, false>(p, st);
    else add ? launch_embedding_few<false, true>(p, st) : launch_embedding_few<false, false>(p, st);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : 1000 + (int)e;
  }
  const EmbLayout at(tokens, rows_local, dim);
  char* s = static_cast<char*>(scratch);
  EmbGrad p = {};
  p.ids = ids;
  p.dout = static_cast<const __nv_bfloat16*>(dout);
  p.dtable = dtable;
  p.range = reinterpret_cast<int2*>(s + at.range);
  p.order = reinterpret_cast<unsigned*>(s + at.order);
  p.valid = reinterpret_cast<int*>(s + at.valid);
  p.taken = p.valid + 1;
  p.codes = reinterpret_cast<unsigned*>(s + at.codes);
  p.part = reinterpret_cast<float*>(s + at.part);
  p.row0 = row0;
  p.tokens = tokens;
  p.rows = rows_local;
  p.dim = dim;
  p.chunk = at.chunk;
  p.share = at.share;
  p.per = emb_per(rows_local);
  p.sets = (rows_local + p.per - 1) / p.per;
  p.shift = 31;
  while (1ll << (p.shift - 31) < p.sets) ++p.shift;
  p.inv = (unsigned)((1ull << p.shift) / p.sets + 1);       // exact for dividends below 2^31
  p.scale = scale;
  const int hists = (EP_WARPS + 1) * p.per * 4, most = (EP_SMEM - hists) / (EP_WARPS * 4);
  p.list = !at.coded || p.share > 1 << 22 ? 0 : p.share < most ? p.share : most;       // (an entry has 22 bits for the token)
  const int smem = hists + EP_WARPS * p.list * 4;
  static std::atomic<unsigned> ready{0};              // a bit for each device
  int device = 0;
  cudaError_t set = cudaGetDevice(&device);
  if (set == cudaSuccess && (device > 31 || !(ready.load(std::memory_order_relaxed) >> device & 1))) {
    set = cudaFuncSetAttribute(embedding_plan_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, EP_SMEM);
    if (set == cudaSuccess) set = cudaFuncSetAttribute(embedding_plan_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, EP_SMEM);
    if (set == cudaSuccess && device <= 31) ready.fetch_or(1u << device, std::memory_order_relaxed);
  }
  if (set != cudaSuccess) return 1000 + (int)set;
  if (at.coded) {
    chain(embedding_code_kernel, (EP_WARPS * p.share + 255) / 256, 256, 0, st, p);
    chain(embedding_plan_kernel<true>, p.sets, EP_WARPS * 32, smem, st, p);
  } else {
    chain(embedding_plan_kernel<false>, p.sets, EP_WARPS * 32, smem, st, p);
  }
  if (dtable_is_f32) add ? launch_embedding_grad<true, true>(p, st) : launch_embedding_grad<true, false>(p, st);
  else add ? launch_embedding_grad<false, true>(p, st) : launch_embedding_grad<false, false>(p, st);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
