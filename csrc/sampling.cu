// The next token of every row of logits, drawn by one given random number a row.
//
// With m the largest logit, w_i = exp((l_i - m) / T).  In the order of the logits, the larger first and of equal ones the lower
// index, the tokens kept are: the first k (top-k), of those the ones with w_i >= min_p, of those the first ones until their weights
// add up to top_p of all that were left (nucleus).  The token drawn is the first, in the order of the indices, at which the sum of the
// kept weights exceeds u times their total.  T = 0 is the first index of the largest logit.  All three filters keep a leading part of
// the order: a smallest logit and how many of that value.
//
// Which token comes out hangs on sums of up to 2^18 weights that are compared with a border, so weights are computed in 64 bits
// (2^x by a table of 2^(j/16) and the series of the rest, 1e-15) and added as whole multiples of 2^-44: sums are exact, and
// the same in any order.
//
// Memory bounds it: a row has to be read once.  A cluster of 1 to 16 CTAs takes a row, each a contiguous slice; more CTAs the fewer
// rows there are.  The first pass over the row finds m and counts the logits by the leading 11 bits of their order; the second, out of L2,
// hands the few that can matter (the bins that hold the first k, those above min_p, the topmost bins) to one CTA, which sorts
// them and finishes alone.  Where they are too many (a flat distribution, many equal logits) the border is found by counting or
// adding up weights over the next bits, pass by pass, and the token in two more.

#include "common.cuh"
#include "tpb.h"

namespace tpb {

int sm_count();

constexpr int SMP_THREADS = 512, SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_BINS = 2048;          // 11 bits of the order at a time: 31-21, 20-10, 9-0
constexpr int SMP_CAP = 2048;           // tokens that one CTA sorts
constexpr int SMP_FIXED = 44;           // a weight of 1 is 2^44: 2^18 of them stay below 2^63

using u64 = unsigned long long;

struct SampleParams {
  const void* logits;
  long long stride;
  const float* u;
  const float *temperature, *top_p, *min_p;      // one a row, or null: the numbers below
  const int* top_k;
  double temperature0, top_p0, min_p0;
  int top_k0, V, slice;                          // slice: logits of a CTA, a multiple of 4
  long long* out;
  int vec;                                       // rows can be read four logits at a time
};

// The place of another CTA's copy of a shared variable.
template <typename T>
__device__ __forceinline__ T* smp_peer(T* p, int rank) {
  u64 a;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"((u64)p), "r"(rank));
  return reinterpret_cast<T*>(a);
}

// Order of the logits as whole numbers: larger logit, larger key; both zeros alike, subnormal ones as they are.
__device__ __forceinline__ unsigned smp_key(float l) {
  unsigned b = __float_as_uint(l);
  if (b == 0x80000000u) b = 0;
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float smp_logit(unsigned key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }

struct SmpWeight {
  double per_unit;        // log2(e) / T
  float top;
  const double* table;    // 2^(j / 16), shared
  __device__ __forceinline__ double real(float l) const {
    if (l == top) return 1.0;
    const double x = ((double)l - (double)top) * per_unit;
    if (!(x > -64.0)) return 0.0;
    const double shifted = fma(x, 16.0, 6755399441055744.0);      // 1.5 * 2^52: the nearest whole number ends up in the low bits
    const int j = __double2loint(shifted);
    const double y = fma(shifted - 6755399441055744.0, -0.0625, x) * 0.6931471805599453;      // |y| <= ln 2 / 32
    double s = fma(y, 1.0 / 720, 1.0 / 120);
    s = fma(s, y, 1.0 / 24);
    s = fma(s, y, 1.0 / 6);
    s = fma(s, y, 0.5);
    s = fma(s, y, 1.0);
    s = fma(s, y, 1.0);
    s *= table[j & 15];
    return __hiloint2double(__double2hiint(s) + ((j >> 4) << 20), __double2loint(s));
  }
  static __device__ __forceinline__ u64 fixed(double w) {         // to the nearest multiple of 2^-44
    return (u64)__double_as_longlong(fma(w, (double)(1LL << SMP_FIXED), 4503599627370496.0)) & 0xfffffffffffffULL;
  }
  __device__ __forceinline__ u64 operator()(float l) const { return fixed(real(l)); }
};

struct SmpShared {
  u64 sums[SMP_BINS];                   // of weights, or counts
  u64 list[SMP_CAP], weight[SMP_CAP];
  double table[16];
  u64 warp[SMP_WARPS], warp2[SMP_WARPS];
  u64 tot[16], tot2[16];                // of the cluster's CTAs
  u64 found[3];                         // bin, sum of the bins above, sum of the bin
  unsigned count;                       // of the list
  int bad;
};

__device__ __forceinline__ u64 smp_warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sum over the block, in every thread.
__device__ __forceinline__ u64 smp_block_sum(u64 v, u64* part) {
  v = smp_warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < SMP_WARPS; ++w) v += part[w];
  return v;
}
// The sum of what the threads before this one have.
__device__ __forceinline__ u64 smp_block_before(u64 v, u64* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  __syncthreads();
  if (lane == 31) part[warp] = sum;
  __syncthreads();
  u64 before = sum - v;
#pragma unroll
  for (int w = 0; w < SMP_WARPS; ++w)
    if (w < warp) before += part[w];
  return before;
}

// All threads of the cluster, which come together warp by warp first (the cluster's barrier is the aligned one).
__device__ __forceinline__ void smp_cluster_sync() {
  __syncthreads();
  cluster_sync_all();
}

// Every CTA's s.sums, added up, from the last bin down: the bin in which the sum reaches `target` (which it does), in s.found.
__device__ __forceinline__ void smp_find(SmpShared& s, u64 target, int rank, int ctas) {
  const int per = SMP_BINS / ctas, b0 = rank * per;
  smp_cluster_sync();
  // four neighbouring bins to a thread, the topmost to thread 0
  u64 v[4] = {}, mine = 0;
  const int high = b0 + per - 1 - (int)threadIdx.x * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (high - i >= b0) {
      for (int c = 0; c < ctas; ++c) v[i] += smp_peer(s.sums, c)[high - i];
      mine += v[i];
    }
  const u64 all = smp_block_sum(mine, s.warp), before = smp_block_before(mine, s.warp);
  if ((int)threadIdx.x < ctas) smp_peer(s.tot, threadIdx.x)[rank] = all;
  smp_cluster_sync();
  u64 above = before;
  for (int c = rank + 1; c < ctas; ++c) above += s.tot[c];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (high - i >= b0 && above < target && above + v[i] >= target)
      for (int c = 0; c < ctas; ++c) {
        u64* f = smp_peer(s.found, c);
        f[0] = high - i;
        f[1] = above;
        f[2] = v[i];
      }
    above += v[i];
  }
  smp_cluster_sync();
}

// s.list[0 .. n) in descending order; n is padded with zeros to a power of two.
__device__ __forceinline__ void smp_sort(u64* list, int n) {
  int size = 32;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += SMP_THREADS) list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int x = threadIdx.x; x < size / 2; x += SMP_THREADS) {
        const int a = 2 * x - (x & (j - 1)), b = a + j;
        const u64 va = list[a], vb = list[b];
        if ((va < vb) == ((a & k) == 0)) {
          list[a] = vb;
          list[b] = va;
        }
      }
      __syncthreads();
    }
}
// s.weight[0 .. n) becomes the sums up to and with each.
__device__ __forceinline__ void smp_scan(SmpShared& s, int n) {
  u64 v[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = threadIdx.x * 4 + i;
    v[i] = x < n ? s.weight[x] : 0;
    mine += v[i];
  }
  u64 sum = smp_block_before(mine, s.warp);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = threadIdx.x * 4 + i;
    sum += v[i];
    if (x < n) s.weight[x] = sum;
  }
  __syncthreads();
}

template <typename L>
__device__ __forceinline__ float smp_read(const L* p);
template <>
__device__ __forceinline__ float smp_read(const float* p) { return *p; }
template <>
__device__ __forceinline__ float smp_read(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Four logits from index i on, -inf for NaN (which is never drawn) and behind `end`.
template <typename L>
__device__ __forceinline__ void smp_load(const L* row, int i, int end, int vec, float* l) {
  if (vec && i + 4 <= end) {
    if constexpr (sizeof(L) == 4) {
      const float4 v = *reinterpret_cast<const float4*>(row + i);
      l[0] = v.x; l[1] = v.y; l[2] = v.z; l[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(row + i);
      const float2 a = unpack_bf16(v.x), b = unpack_bf16(v.y);
      l[0] = a.x; l[1] = a.y; l[2] = b.x; l[3] = b.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) l[e] = i + e < end ? smp_read<L>(row + i + e) : -INFINITY;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) l[e] = l[e] != l[e] ? -INFINITY : l[e];
}
// f(index, logits, how many) for the CTA's slice, four at a time.
template <typename L, typename F>
__device__ __forceinline__ void smp_stream(const L* row, int begin, int end, int vec, F&& f) {
  constexpr int AHEAD = 4, STEP = SMP_THREADS * 4;
  for (int i0 = begin; i0 < end; i0 += AHEAD * STEP) {
    float l[AHEAD][4];
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) {
      const int i = i0 + x * STEP + threadIdx.x * 4;
      if (i < end) smp_load<L>(row, i, end, vec, l[x]);
    }
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) {
      const int i = i0 + x * STEP + threadIdx.x * 4;
      f(i, l[x], min(4, end - i));      // (none: 0 or less)
    }
  }
}

template <typename L>
__global__ void __launch_bounds__(SMP_THREADS, 2)
sample_kernel(const SampleParams p, int ctas) {
  if (!chain_begin()) return;
  extern __shared__ __align__(16) uint8_t smp_smem[];
  SmpShared& s = *reinterpret_cast<SmpShared*>(smp_smem);
  const int rank = ctas > 1 ? (int)cluster_ctarank() : 0, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / ctas, V = p.V;
  const L* row = static_cast<const L*>(p.logits) + b * p.stride;
  const int begin = min(V, rank * p.slice), end = min(V, begin + p.slice);
  const double T = p.temperature ? (double)p.temperature[b] : p.temperature0;
  double top_p = p.top_p ? (double)p.top_p[b] : p.top_p0, min_p = p.min_p ? (double)p.min_p[b] : p.min_p0;
  int top_k = p.top_k ? p.top_k[b] : p.top_k0;
  const bool greedy = !(T > 0.0);
  if (top_k <= 0 || top_k >= V) top_k = 0;
  const bool nucleus = top_p < 1.0;               // (NaN: off)
  top_p = fmax(top_p, 0.0);
  min_p = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
  const bool count = !greedy && (top_k || nucleus || min_p > 0.0);
  for (int i = tid; i < SMP_BINS; i += SMP_THREADS) s.sums[i] = 0;
  if (tid < 16) s.table[tid] = exp2(tid * 0.0625);
  if (tid == 0) s.count = 0, s.bad = 0;
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (nobody writes to a CTA that has not begun)
  unsigned* const counts = reinterpret_cast<unsigned*>(s.sums);   // the low halves (little-endian) of the sums

  // ---- the largest logit, its first index, and how many logits there are in each bin
  unsigned top_key = 0;
  int at = V;
  smp_stream<L>(row, begin, end, p.vec, [&](int i, const float* l, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) {
        const unsigned key = smp_key(l[e]);
        if (key > top_key) top_key = key, at = i + e;
        if (count) atomicAdd(counts + 2 * (key >> 21), 1u);
      }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned x = __shfl_xor_sync(0xffffffffu, top_key, o);
    const int y = __shfl_xor_sync(0xffffffffu, at, o);
    if (x > top_key || (x == top_key && y < at)) top_key = x, at = y;
  }
  if (lane == 0) s.warp[warp] = (u64)top_key << 32 | (unsigned)(V - at);
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid < ctas) {
    u64 best = 0;
    for (int w = 0; w < SMP_WARPS; ++w) best = max(best, s.warp[w]);
    smp_peer(s.tot2, tid)[rank] = best;
  }
  smp_cluster_sync();
  u64 best = 0;
  for (int c = 0; c < ctas; ++c) best = max(best, s.tot2[c]);
  const float top = smp_logit((unsigned)(best >> 32));
  at = V - (int)(unsigned)best;
  if (greedy || top == -INFINITY) {
    if (rank == 0 && tid == 0) p.out[b] = top == -INFINITY ? -1 : at;
    return;
  }
  const SmpWeight weight = {1.4426950408889634 / T, top, s.table};
  const double u = fmin(fmax((double)p.u[b], 0.0), 1.0);
  auto place = [&](u64 total) {                   // the sum that the drawn token's passes
    const u64 x = (u64)(u * (double)total);
    return x < total ? x : total - 1;
  };

  unsigned border = 0;                            // smallest key kept, and how many of it
  u64 of_border = 0;
  bool few = count;
  if (count) {
    // ---- the bins that can matter
    const bool all_fit = !top_k && V <= SMP_CAP;
    unsigned lowest = 0;                          // bin
    if (!all_fit) {
      smp_find(s, top_k ? top_k : SMP_CAP + 1, rank, ctas);
      if (top_k) {
        lowest = (unsigned)s.found[0];
        few = s.found[1] + s.found[2] <= SMP_CAP;
      } else {
        lowest = (unsigned)s.found[0] + 1;
      }
    }
    if (!top_k && min_p > 0.0) {
      float least = __double2float_rd((double)top + log(min_p) * T * (1.0 + 1e-12));
      if (!(least == least)) least = -INFINITY;               // (T is infinite)
      if (fabsf(least) < 1.2e-38f) least = -1.2e-38f;         // (subnormal)
      const unsigned bin = smp_key(least) >> 21;
      if (bin < lowest) few = false;
      else lowest = bin;
    }
    if (few) {
      const bool need_total = nucleus && !top_k && !(min_p > 0.0);
      u64 total = 0;
      u64* const list = smp_peer(s.list, 0);
      unsigned* const n_list = smp_peer(&s.count, 0);
      smp_stream<L>(row, begin, end, p.vec, [&](int i, const float* l, int n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned key = smp_key(l[e]);
          const bool mine = e < n && key >> 21 >= lowest;
          if (mine) {
            const unsigned x = atomicAdd(n_list, 1u);
            if (x < SMP_CAP) list[x] = (u64)key << 32 | (0xffffffffu - (unsigned)(i + e));
          }
          if (need_total && e < n) total += weight(l[e]);
        }
      });
      if (need_total) {
        total = smp_block_sum(total, s.warp);
        if (tid == 0) smp_peer(s.tot, 0)[rank] = total;
      }
      smp_cluster_sync();
      if (rank == 0) {
        // ---- one CTA sorts them and finishes
        const int n = min(s.count, (unsigned)SMP_CAP);
        smp_sort(s.list, n);
        int kept = top_k ? min(n, top_k) : n;
        u64 below = 0;                            // (counts of this thread's)
        for (int i = tid; i < n; i += SMP_THREADS) {
          const double w = weight.real(smp_logit((unsigned)(s.list[i] >> 32)));
          s.weight[i] = SmpWeight::fixed(w);
          below += i < kept && w < min_p;
        }
        kept -= (int)smp_block_sum(below, s.warp);
        smp_scan(s, n);
        u64 sum = kept > 0 ? s.weight[kept - 1] : 0;
        if (need_total) {
          sum = 0;
          for (int c = 0; c < ctas; ++c) sum += s.tot[c];
        }
        if (nucleus) {
          const u64 border_sum = __double2ull_ru(top_p * (double)sum);
          u64 in = 0;
          for (int i = tid; i < kept; i += SMP_THREADS) in += i == 0 || s.weight[i - 1] < border_sum;
          const int inside = (int)smp_block_sum(in, s.warp);
          if (need_total && inside == n && (n == 0 || s.weight[n - 1] < border_sum)) {
            if (tid < ctas) *smp_peer(&s.bad, tid) = 1;           // the border lies below the list
          }
          kept = inside;
          __syncthreads();
        }
        if (!s.bad) {
          const u64 target = place(s.weight[kept - 1]);
          __syncthreads();
          for (int i = tid; i < kept; i += SMP_THREADS) {
            const u64 x = s.list[i];
            s.list[i] = x << 32 | x >> 32;        // by index now
          }
          smp_sort(s.list, kept);
          for (int i = tid; i < kept; i += SMP_THREADS) s.weight[i] = weight(smp_logit((unsigned)s.list[i]));
          __syncthreads();
          smp_scan(s, kept);
          for (int i = tid; i < kept; i += SMP_THREADS)
            if (s.weight[i] > target && (i == 0 || s.weight[i - 1] <= target)) p.out[b] = 0xffffffffu - (unsigned)(s.list[i] >> 32);
        }
      }
      if (!need_total) return;
      smp_cluster_sync();
      if (!s.bad) return;
    }

    // ---- the border by the rest of the order's bits
    auto refine = [&](bool weights, u64 target, unsigned known, int from) {      // bits below `from` of the border's key
      u64 above = 0;
      for (int shift = from == 32 ? 21 : from == 21 ? 10 : 0;;) {
        const int bits = shift == 21 ? 11 : shift == 10 ? 11 : 10;
        __syncthreads();
        for (int i = tid; i < SMP_BINS; i += SMP_THREADS) s.sums[i] = 0;
        __syncthreads();
        smp_stream<L>(row, begin, end, p.vec, [&](int i, const float* l, int n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned key = smp_key(l[e]);
            if (e >= n || (shift < 21 && key >> (shift + bits) != known >> (shift + bits))) continue;
            const unsigned bin = key >> shift & ((1u << bits) - 1);
            if (!weights) {
              atomicAdd(counts + 2 * bin, 1u);
            } else if (key > border) {
              const double w = weight.real(l[e]);
              const u64 f = SmpWeight::fixed(w);
              if (w >= min_p && f) atomicAdd(s.sums + bin, f);
            }
          }
        });
        smp_find(s, target - above, rank, ctas);
        known |= (unsigned)s.found[0] << shift;
        above += s.found[1];
        if (shift == 0) break;
        shift = shift == 21 ? 10 : 0;
      }
      of_border = above;                          // what lies above it
      return known;
    };
    if (top_k) {
      const u64 above = s.found[1];
      border = refine(false, top_k - above, (unsigned)s.found[0] << 21, 21);
      of_border = top_k - above - of_border;
    }
    if (nucleus) {
      // all that is left so far
      u64 total = 0;
      smp_stream<L>(row, begin, end, p.vec, [&](int i, const float* l, int n) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < n && smp_key(l[e]) > border) {
            const double w = weight.real(l[e]);
            if (w >= min_p) total += SmpWeight::fixed(w);
          }
      });
      total = smp_block_sum(total, s.warp);
      if (tid < ctas) smp_peer(s.tot2, tid)[rank] = total;
      smp_cluster_sync();
      total = 0;
      for (int c = 0; c < ctas; ++c) total += s.tot2[c];
      u64 each = 0;
      if (top_k) {
        const double w = weight.real(smp_logit(border));
        if (w >= min_p) each = SmpWeight::fixed(w);
      }
      const u64 want = max(__double2ull_ru(top_p * (double)(total + each * of_border)), 1ULL);
      if (want > total && each) {
        of_border = min(of_border, (want - total + each - 1) / each);
      } else {
        const unsigned key = refine(true, min(want, total), 0, 32);
        const u64 w = weight(smp_logit(key));
        of_border = (min(want, total) - of_border + w - 1) / w;
        border = key;
      }
    }
  }

  // ---- the token: sums of the slices, of the warps' parts of the one it lies in, then along that part
  const u64 each = border ? [&] { const double w = weight.real(smp_logit(border)); return w >= min_p ? SmpWeight::fixed(w) : 0; }() : 0;
  const int part = ((end - begin + SMP_WARPS - 1) / SMP_WARPS + 127) / 128 * 128;
  const int from = min(end, begin + warp * part), to = min(end, from + part);
  auto add = [&](int i, u64& sum, u64& equal) {   // four logits of a lane
    float l[4];
    if (i < to) smp_load<L>(row, i, to, p.vec && (from & 3) == 0, l);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < to) {
        const unsigned key = smp_key(l[e]);
        if (key > border) {
          const double w = weight.real(l[e]);
          if (w >= min_p) sum += SmpWeight::fixed(w);
        } else if (key == border) {
          ++equal;
        }
      }
  };
  u64 sum = 0, equal = 0;
#pragma unroll 2
  for (int i = from + lane * 4; i < to; i += 128) add(i, sum, equal);
  sum = smp_warp_sum(sum);
  equal = smp_warp_sum(equal);
  __syncthreads();
  if (lane == 0) s.warp[warp] = sum, s.warp2[warp] = equal;
  __syncthreads();
  if (tid < ctas) {
    u64 x = 0, y = 0;
    for (int w = 0; w < SMP_WARPS; ++w) x += s.warp[w], y += s.warp2[w];
    smp_peer(s.tot, tid)[rank] = x;
    smp_peer(s.tot2, tid)[rank] = y;
  }
  smp_cluster_sync();
  auto upto = [&](u64 x, u64 y) { return x + each * min(y, of_border); };
  u64 x = 0, y = 0;
  for (int c = 0; c < ctas; ++c) x += s.tot[c], y += s.tot2[c];
  const u64 target = place(upto(x, y));
  x = y = 0;
  for (int c = 0; c < rank; ++c) x += s.tot[c], y += s.tot2[c];
  for (int w = 0; w < warp; ++w) x += s.warp[w], y += s.warp2[w];
  if (upto(x, y) > target || upto(x + sum, y + equal) <= target) return;
  for (int i0 = from; i0 < to; i0 += 128) {
    u64 mine = 0, ties = 0;
    add(i0 + lane * 4, mine, ties);
    const u64 all = smp_warp_sum(mine), all_ties = smp_warp_sum(ties);
    if (upto(x + all, y + all_ties) > target) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 a = __shfl_up_sync(0xffffffffu, mine, o), c = __shfl_up_sync(0xffffffffu, ties, o);
        if (lane >= o) mine += a, ties += c;
      }
      const unsigned past = __ballot_sync(0xffffffffu, upto(x + mine, y + ties) > target);
      const int owner = __ffs(past) - 1;
      u64 before = __shfl_up_sync(0xffffffffu, mine, 1), before_ties = __shfl_up_sync(0xffffffffu, ties, 1);
      if (lane == 0) before = before_ties = 0;
      if (lane == owner) {
        const int i = i0 + lane * 4;
        float l[4];
        smp_load<L>(row, i, to, 0, l);
        u64 a = x + before, c = y + before_ties;
        for (int e = 0; e < 4 && i + e < to; ++e) {
          const unsigned key = smp_key(l[e]);
          if (key > border) {
            const double w = weight.real(l[e]);
            if (w >= min_p) a += SmpWeight::fixed(w);
          } else if (key == border) {
            ++c;
          }
          if (upto(a, c) > target) {
            p.out[b] = i + e;
            break;
          }
        }
      }
      return;
    }
    x += all;
    y += all_ties;
  }
}

template <typename L>
static int launch_sample(const SampleParams& p, int B, int ctas, cudaStream_t stream) {
  auto* f = sample_kernel<L>;
  cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SmpShared));
  if (e == cudaSuccess && ctas > 8) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = chain_clusters(f, ctas, dim3(B * ctas), SMP_THREADS, sizeof(SmpShared), stream, p, ctas);
  const cudaError_t last = cudaGetLastError();
  if (e == cudaSuccess) e = last;
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

}  // namespace tpb

using namespace tpb;

// out [B] (int64): the token drawn from row b of logits [B, V] (fp32, or bf16; rows `stride` apart) by u[b] in [0, 1); -1 for a row
// without a logit above -inf.  temperature, top_p, min_p (fp32) and top_k (int32): one a row in device memory, or null for the
// numbers behind them.  V up to 2^18.
extern "C" int tpb_sample_tokens(const void* logits, int bf16, long long stride, const float* u, const float* temperature,
                                 const int* top_k, const float* top_p, const float* min_p, double temperature0, int top_k0,
                                 double top_p0, double min_p0, long long* out, int B, int V, void* stream_) {
  if (B < 0 || V < 1 || V > (1 << 18)) return -2;
  if (B == 0) return 0;
  if (B > (0x7fffffff >> 4)) return -2;
  // As many CTAs to a row as keep the machine busy, with 2048 logits or more each.
  int ctas = 1;
  while (ctas < 16 && (long long)B * ctas * 2 <= 4LL * sm_count() && V / (ctas * 2) >= 2048) ctas *= 2;
  const int elt = bf16 ? 2 : 4;
  SampleParams p = {logits, stride, u, temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0, V,
                    ((V + ctas - 1) / ctas + 3) / 4 * 4, out, 0};
  p.vec = reinterpret_cast<uintptr_t>(logits) % (4 * elt) == 0 && stride % 4 == 0;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return bf16 ? launch_sample<__nv_bfloat16>(p, B, ctas, stream) : launch_sample<float>(p, B, ctas, stream);
}
