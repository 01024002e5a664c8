// The next token of every row of logits, drawn by one given random number a row.
//
// With m the largest logit, w_i = exp((l_i - m) / T).  In the order of the logits, the larger first and of equal ones the lower
// index, the tokens kept are: the first k (top-k), of those the ones with w_i >= min_p, of those the first ones until their weights
// add up to top_p of all that were left (nucleus).  The token drawn is the first, in the order of the indices, at which the sum of the
// kept weights exceeds u times their total.  T = 0 is the first index of the largest logit.  All three filters keep a leading part of
// the order: a smallest logit and how many of that value.
//
// Which token comes out hangs on sums of up to 2^18 weights that are compared with a border, so fp32 exponentials will not do: a
// weight is a table's 2^(j / 1024) times the series of the rest, with the exponent as an unevaluated sum of two floats, good to 2^-34
// (in fp64 throughout, an early form took five times as long for 65 M weights), and weights are added as whole multiples of 2^-44: sums are
// exact, and the same in any order.
//
// Memory bounds it: a row has to be read once.  A cluster of 1 to 16 CTAs takes a row, each a contiguous slice; more CTAs the fewer
// rows there are.  A slice comes through a ring of bulk copies, or stays in it where it fits.
//   * The first pass finds m.
//   * top-k: the k-th largest of the threads' own largest logits is a lower bound of the k-th largest of all; min-p has a bound of its
//     own.  The logits from the bound on, usually little more than k, go to one CTA, which sorts them and finishes alone.  A long slice
//     with a small k has them staged by the first pass.
//   * nucleus: a histogram of the weights over their exponents in steps of 1/64; the bin with the border goes to one CTA, which
//     sorts it.  Then two more passes draw the token: sums of slices and of the parts of their warps, and along one of those.
//   * Where a list is too long for one CTA (thousands of equal logits, large k) the border is found bit by bit of the order.

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "tpb.h"

namespace tpb {

constexpr int SMP_THREADS = 512, SMP_WARPS = SMP_THREADS / 32;      // (1024, when one row's nucleus took 36 us instead of 33: 41)
constexpr int SMP_BINS = 2048;          // 11 bits of the order at a time (31-21, 20-10, 9-0); 32 binary orders of weights in steps of 1/64
constexpr int SMP_CAP = 2048;           // tokens that one CTA sorts
constexpr int SMP_FEW = SMP_THREADS / 4;        // largest k whose candidates are found while a row is read
constexpr int SMP_FIXED = 44;           // a weight of 1 is 2^44: 2^18 of them stay below 2^63
constexpr int SMP_TABLE = 1024;         // 2^(j / 1024)
constexpr int SMP_CHUNK = SMP_THREADS * 8, SMP_RING = 3;       // logits of a bulk copy, copies under way

using u64 = unsigned long long;

// 2^62 2^(j / 1024), to a double's precision.
struct SmpTable {
  u64 at[SMP_TABLE];
  constexpr SmpTable() : at() {
    for (int j = 0; j < SMP_TABLE; ++j) {
      const double y = j * (0.69314718055994530942 / SMP_TABLE);
      double sum = 1, term = 1;
      for (int k = 1; k < 24; ++k) {
        term *= y / k;
        sum += term;
      }
      at[j] = (u64)(sum * 4611686018427387904.0);
    }
  }
};
__device__ const SmpTable smp_table = SmpTable();

struct SampleParams {
  const void* logits;
  long long stride;
  const float* u;
  const float *temperature, *top_p, *min_p;      // one a row, or null: the numbers below
  const int* top_k;
  double temperature0, top_p0, min_p0;
  int top_k0, B, V, slice;                       // slice: logits of a CTA of several, a multiple of 8
  int unequal, whole;                            // rows take unequal times; of them, how many take a whole cluster, the others a CTA each
                                                 // (0: every row takes a cluster)
  long long* out;
  int vec;                                       // rows can be read four logits at a time: 2, also by bulk copies (16-byte aligned)
  int* status;
};

// The place of another CTA's copy of a shared variable.
template <typename T>
__device__ __forceinline__ T* smp_peer(T* p, int rank) {
  u64 a;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"((u64)p), "r"(rank));
  return reinterpret_cast<T*>(a);
}

// A logit as it counts: -inf for NaN, 0 for -0; subnormal ones as they are (this file is compiled to flush them in fp32 arithmetic).
__device__ __forceinline__ float smp_clean(float l) {
  asm("max.f32 %0, %0, 0fFF800000;\n\tadd.rn.f32 %0, %0, 0f00000000;" : "+f"(l));
  return l;
}
// Order of the logits as whole numbers: larger logit, larger key.
__device__ __forceinline__ unsigned smp_key(float l) {
  const int b = __float_as_int(smp_clean(l));
  return (unsigned)(b ^ (b >> 31 | (int)0x80000000));
}
// The largest of four logits (no NaN, unless all are).
__device__ __forceinline__ float smp_max4(const float* l) {
  float m;
  asm("max.f32 %0, %1, %2;\n\tmax.f32 %0, %0, %3;\n\tmax.f32 %0, %0, %4;" : "=&f"(m) : "f"(l[0]), "f"(l[1]), "f"(l[2]), "f"(l[3]));
  return m;
}
__device__ __forceinline__ float smp_logit(unsigned key) { return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xffffffffu)); }

// To 64 bits, with subnormal numbers.
__device__ __forceinline__ double smp_double(float a) {
  double r;
  asm("cvt.f64.f32 %0, %1;" : "=d"(r) : "f"(a));
  return r;
}
// Larger, and the same, in that order, with subnormal numbers.
__device__ __forceinline__ bool smp_above(float a, float b) {
  int x;
  asm("{\n\t.reg .pred p;\n\tsetp.gt.f32 p, %1, %2;\n\tselp.s32 %0, 1, 0, p;\n\t}" : "=r"(x) : "f"(a), "f"(b));
  return x;
}
__device__ __forceinline__ bool smp_same(float a, float b) {
  int x;
  asm("{\n\t.reg .pred p;\n\tsetp.eq.f32 p, %1, %2;\n\tselp.s32 %0, 1, 0, p;\n\t}" : "=r"(x) : "f"(a), "f"(b));
  return x;
}

struct SmpWeight {
  double per_unit;        // log2(e) / T
  float hi, lo;           // 1024 log2(e) / T as a sum of two floats
  const u64* table;       // 2^62 2^(j / 1024), shared
  float top;              // the largest logit
  float p_top, p_cut;     // 1024 log2 of the largest weight, and 2^-45 of it, before that is made 1: the nearest product
  int j_top;              // the whole number it is nearest to (with the other bits of the pattern), and what is missing
  float y_top;
  bool slow;              // T, or the logits, too far from 1 for that: 64 bits

  __device__ __forceinline__ SmpWeight(double T, const u64* table_) : per_unit(1.4426950408889634 / T), table(table_) {
    const double c = per_unit * SMP_TABLE;
    hi = (float)c;
    lo = (float)(c - (double)hi);
    slow = !(T > 1e-20 && T < 1e20);
  }
  __device__ __forceinline__ void begin(float top_) {
    top = top_;
    slow |= !(fabsf(top) * hi < 2097152.f);
    p_top = __fmul_rn(top, hi);
    p_cut = p_top - 45.f * SMP_TABLE;
    split(top, p_top, 0.f, j_top, y_top);
  }
  // 1024 l log2(e) / T = j + y, j whole (in the low bits of a float's pattern), less y0; p = l * hi
  __device__ __forceinline__ void split(float l, float p, float y0, int& j, float& y) const {
    const float shifted = __fadd_rn(p, 12582912.f);             // 1.5 * 2^23 (not as one fma: step() has to see the same)
    j = __float_as_int(shifted);
    y = (p - (shifted - 12582912.f)) + (fmaf(l, hi, -p) + fmaf(l, lo, -y0));
  }
  // in 64 bits
  __device__ __noinline__ double real(float l) const {
    const double x = (smp_double(l) - smp_double(top)) * per_unit;
    return smp_same(l, top) ? 1.0 : x > -100.0 ? exp2(x) : 0.0;         // (NaN, of infinities: 0)
  }
  __device__ __noinline__ int step_slow(float l) const {
    return smp_same(l, top) ? 0 : (int)fmax(fmin(rint((smp_double(l) - smp_double(top)) * per_unit * SMP_TABLE), 0.0), -1e9);
  }
  // 1024 log2 of the weight, rounded: does not fall where l grows.
  __device__ __forceinline__ int step(float l) const {
    return slow ? step_slow(l) : __float_as_int(__fadd_rn(fmaxf(__fmul_rn(l, hi), p_cut), 12582912.f)) - j_top;
  }
  // In multiples of 2^-44: 2^44 for the largest, else with the last bit set, as often above as below what is cut off; 0 below 2^-45 and
  // for NaN and where it is not wanted.  j: step(l).
  template <bool SLOW>
  __device__ __forceinline__ u64 of(float l, int& j, bool wanted = true) const {
    if (SLOW) {
      j = step_slow(l);
      return wanted ? __double2ull_rn(real(l) * (double)(1LL << SMP_FIXED)) : 0;
    }
    const float p = __fmul_rn(l, hi);
    float y;
    split(l, fmaxf(p, p_cut), y_top, j, y);
    j -= j_top;
    y *= 0.69314718056f / SMP_TABLE;
    const float q = fmaf(fmaf(y, 1.f / 6, 0.5f) * y, y, y);     // 2^rest - 1, |q| < 2^-10; the next term is below 2^-46
    const int qi = __float_as_int(q + 0.0029296875f) - 0x3b400000;       // 1.5 * 2^-9: in multiples of 2^-32
    const u64 t = table[j & (SMP_TABLE - 1)];
    const u64 w = t + (u64)((long long)(int)(t >> 32) * qi);
    const u64 x = w >> (62 - SMP_FIXED - (j >> 10));
    return wanted & (p > p_cut) ? x | (~x >> SMP_FIXED & 1) : 0;
  }
  __device__ __forceinline__ u64 operator()(float l) const {
    int j;
    return slow ? of<true>(l, j) : of<false>(l, j);
  }
  // f(std::true_type) where weights are slow, else f(std::false_type)
  template <typename F>
  __device__ __forceinline__ void either(F&& f) const {
    if (slow) f(std::true_type());
    else f(std::false_type());
  }
  // Steps of 1/64 below the largest weight's exponent, the largest weights in the last bin, all below 2^-32 in the first.
  static __device__ __forceinline__ int bin(int j) { return SMP_BINS - 1 + max(j >> 4, 1 - SMP_BINS); }
};

// The smallest key in (low, high] for which `past` holds, as it does for `high` and for all behind; the whole warp calls.
template <typename F>
__device__ __forceinline__ unsigned smp_first_key(unsigned low, unsigned high, F&& past) {
  while (high - low > 1) {
    const unsigned wide = (high - low + 32) / 33, at = low + wide * ((threadIdx.x & 31) + 1);
    const unsigned which = __ballot_sync(0xffffffffu, at >= high || past(at));
    const int n = which ? __ffs(which) - 1 : 32;                // lanes in front of the border
    high = min(high, low + wide * (n + 1));
    low += wide * n;
  }
  return high;
}
constexpr unsigned SMP_LOWEST = 0x007fffffu, SMP_HIGHEST = 0xff800000u;      // keys of -inf and inf

struct SmpShared {
  float ring[SMP_RING * SMP_CHUNK];     // bf16 logits take half of it
  u64 sums[SMP_BINS];                   // of weights, or counts
  u64 list[SMP_CAP], weight[SMP_CAP];
  u64 table[SMP_TABLE];
  u64 warp[SMP_WARPS], warp2[SMP_WARPS];
  u64 tops[16], tot[16], ties[16];      // of the cluster's CTAs: largest logits, sums, equal logits.  (Not one array for the first and the
                                        // last: a row without a filter meets no barrier of the cluster between them)
  unsigned bounds[16];                  // the same: all that belongs to the list is staged from there on; 0: it is not
  uint64_t full[SMP_RING];              // barriers of the copies
  u64 found[3];                         // bin, sum of the bins above, sum of all
  unsigned border, of_border;
  unsigned range[2];                    // of keys
  int row;
  unsigned staged, listed;              // tokens of this CTA that may belong to the list, and that do
  int dead;                             // a copy has not come
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

// The CTAs that share a row: a cluster, or one CTA of it.
struct SmpGroup {
  int first, rank, ctas;
  template <typename T>
  __device__ __forceinline__ T* peer(T* p, int of) const { return smp_peer(p, first + of); }
  // All threads, which come together warp by warp first (the cluster's barrier is the aligned one).
  __device__ __forceinline__ void sync() const {
    __syncthreads();
    if (ctas > 1) cluster_sync_all();
  }
};

// Every CTA's s.sums, added up, from the last bin down: the bin in which the sum reaches target(sum of all), in s.found; the
// sum of all alone where that is more.  (s.list and s.weight are used.)
template <typename F>
__device__ __forceinline__ void smp_find(SmpShared& s, const SmpGroup& group, F&& target) {
  const int rank = group.rank, ctas = group.ctas, per = SMP_BINS / ctas, b0 = rank * per, tid = threadIdx.x;
  const u64* total = s.sums;
  if (ctas > 1) {                       // each CTA adds up its share of the bins, for all
    group.sync();
    const int groups = max(1, min(SMP_THREADS / per, ctas));
    for (int x = tid; x < per * groups; x += SMP_THREADS) {
      u64 sum = 0;
#pragma unroll 4
      for (int c = x / per; c < ctas; c += groups) sum += group.peer(s.sums, c)[b0 + x % per];
      s.weight[x] = sum;
    }
    __syncthreads();
    for (int x = tid; x < per * ctas; x += SMP_THREADS) {
      u64 sum = 0;
      for (int g = 0; g < groups; ++g) sum += s.weight[g * per + x % per];
      group.peer(s.list, x / per)[b0 + x % per] = sum;
    }
    group.sync();
    total = s.list;
  } else {
    __syncthreads();
  }
  constexpr int N = SMP_BINS / SMP_THREADS;     // neighbouring bins to a thread, the topmost to thread 0
  u64 v[N], mine = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) mine += v[i] = total[SMP_BINS - 1 - (tid * N + i)];
  u64 above = smp_block_before(mine, s.warp), all = 0;
#pragma unroll
  for (int w = 0; w < SMP_WARPS; ++w) all += s.warp[w];
  const u64 t = target(all);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (above < t && above + v[i] >= t) s.found[0] = SMP_BINS - 1 - (tid * N + i), s.found[1] = above;
    above += v[i];
  }
  if (tid == 0) s.found[2] = all;
  __syncthreads();
}

// s.list[0 .. n) in descending order: no two are the same.  Few go to where the larger ones leave them room; more are padded with zeros
// to a power of two and merged.
__device__ __forceinline__ void smp_sort(u64* list, int n) {
  if (n <= SMP_THREADS) {
    __syncthreads();
    const u64 mine = (int)threadIdx.x < n ? list[threadIdx.x] : 0;
    int larger = 0;
    if ((int)threadIdx.x < n) {
#pragma unroll 8
      for (int i = 0; i < n; ++i) larger += list[i] > mine;
    }
    __syncthreads();
    if ((int)threadIdx.x < n) list[larger] = mine;
    __syncthreads();
    return;
  }
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
  constexpr int N = SMP_CAP / SMP_THREADS;
  u64 v[N], mine = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int x = threadIdx.x * N + i;
    mine += v[i] = x < n ? s.weight[x] : 0;
  }
  u64 sum = smp_block_before(mine, s.warp);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int x = threadIdx.x * N + i;
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

// Four logits from index i on, -inf behind `end`.
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
}

// The CTA's slice, pass by pass.
template <typename L>
struct SmpSlice {
  const L* row;
  int begin, end, vec;
  int copied;                           // what bulk copies can bring ends here: whole 16 bytes
  bool kept = false;                    // all of it lies in the ring
  bool alive = true;                    // no copy has failed to come
  unsigned parity = 0;                  // of the ring's barriers, a bit each

  __device__ __forceinline__ void copy(SmpShared& s, int chunk) const {       // one thread
    const int at = begin + chunk * SMP_CHUNK, n = min(SMP_CHUNK, copied - at) * (int)sizeof(L), slot = chunk % SMP_RING;
    fence_proxy_async();                // (what the block has read of the slot, ahead of the copy that overwrites it)
    mbar_expect_tx(&s.full[slot], max(n, 0));
    if (n > 0)
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                   :
                   : "r"(smem_u32(reinterpret_cast<L*>(s.ring) + slot * SMP_CHUNK)), "l"(row + at), "r"(n), "r"(smem_u32(&s.full[slot]))
                   : "memory");
  }
  __device__ __forceinline__ bool streams() const { return vec == 2 && end - begin > SMP_RING * SMP_CHUNK; }
  // f(index, four logits) for all of them; -inf stands behind the end of the row
  template <typename F>
  __device__ __forceinline__ void pass(SmpShared& s, int* status, F&& f) {
    pass(s, status, f, [](int, auto&&) {});
  }
  // Where it streams, between(chunk, sweep) follows each chunk, and sweep(g) goes over that chunk again.
  template <typename F, typename G>
  __device__ __forceinline__ void pass(SmpShared& s, int* status, F&& f, G&& between) {
    const int chunks = (end - begin + SMP_CHUNK - 1) / SMP_CHUNK, tid = threadIdx.x;
    if (vec < 2) {
      for (int i0 = begin; i0 < end; i0 += SMP_CHUNK) {
        float l[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int i = i0 + (x * SMP_THREADS + tid) * 4;
          if (i < end) smp_load<L>(row, i, end, vec, l[x]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int i = i0 + (x * SMP_THREADS + tid) * 4;
          if (i < end) f(i, l[x]);
        }
      }
      return;
    }
    if (!kept) {
      __syncthreads();
      if (tid == 0 && alive)
        for (int c = 0; c < min(chunks, SMP_RING); ++c) copy(s, c);
    }
    for (int c = 0, slot = 0; c < chunks; ++c) {
      if (!kept) {
        if (alive && !mbar_wait(&s.full[slot], parity >> slot & 1, status, kTimeoutTmaFull, 76)) {
          alive = false;
          s.dead = 1;
        }
        parity ^= 1u << slot;
      }
      const L* ring = reinterpret_cast<const L*>(s.ring) + slot * SMP_CHUNK;
      const int at = begin + c * SMP_CHUNK;
      auto sweep = [&](auto&& g) {
        if (at + SMP_CHUNK <= copied) {
          float l[2][4];
#pragma unroll
          for (int x = 0; x < 2; ++x) smp_load<L>(ring, (x * SMP_THREADS + tid) * 4, SMP_CHUNK, 1, l[x]);
#pragma unroll
          for (int x = 0; x < 2; ++x) g(at + (x * SMP_THREADS + tid) * 4, l[x]);
        } else {
          for (int in = tid * 4; at + in < end && in < SMP_CHUNK; in += SMP_THREADS * 4) {
            float l[4];
            if (at + in + 4 <= copied) smp_load<L>(ring, in, SMP_CHUNK, 1, l);
            else smp_load<L>(row, at + in, end, 0, l);
            g(at + in, l);
          }
        }
      };
      sweep(f);
      between(c, sweep);
      if (!kept && chunks > SMP_RING) {
        __syncthreads();
        if (tid == 0 && alive && c + SMP_RING < chunks) copy(s, c + SMP_RING);
      }
      if (++slot == SMP_RING) slot = 0;
    }
    kept = chunks <= SMP_RING;
  }
};

template <typename L>
__global__ void __launch_bounds__(SMP_THREADS, 1024 / SMP_THREADS)
sample_kernel(const SampleParams p, int ctas) {
  extern __shared__ __align__(128) uint8_t smp_smem[];
  SmpShared& s = *reinterpret_cast<SmpShared*>(smp_smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < SMP_RING) mbar_init(&s.full[tid], 1);
  if (tid == 0) s.dead = 0, s.row = -1;
  fence_barrier_init();
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");      // (nobody writes to a CTA that has not begun)
  chain_launch();
  if (!chain_wait()) return;
  const int V = p.V;
  int b = blockIdx.x / ctas;
  SmpGroup group = {0, ctas > 1 ? (int)cluster_ctarank() : 0, ctas};
  if (p.unequal) {
    // Rows in order of how long they take: those whose sums take all their logits; those that may, with more tokens than a list holds;
    // those with a small k; greedy ones.  The first two kinds get the whole clusters that there are.  Rows of a kind are numbered thread
    // by thread, in quarters of 64 bits.  (In the batch's order: 123 us instead of 114, in the form that gave every row two CTAs.)
    auto kind = [&](int i) {
      const int k = p.top_k ? p.top_k[i] : p.top_k0;
      if (!((p.temperature ? smp_double(p.temperature[i]) : p.temperature0) > 0.0)) return 48;
      if (k > 0 && k <= SMP_FEW) return 32;
      return (k > 0 && k < V) || (p.min_p ? smp_double(p.min_p[i]) : p.min_p0) > 0.0 ? 16 : 0;
    };
    u64 mine = 0, all = 0;
    for (int i = tid; i < p.B; i += SMP_THREADS) mine += 1ULL << kind(i);
    u64 at = smp_block_before(mine, s.warp);
    for (int w = 0; w < SMP_WARPS; ++w) all += s.warp[w];
    const u64 begins = (all << 16) + (all << 32) + (all << 48);
    at += begins;
    const int whole = p.whole ? min((int)(begins >> 32 & 0xffff), p.whole) : p.B;
    if (b >= whole) {
      b = whole + (b - whole) * ctas + group.rank;
      group = {group.rank, 0, 1};
    }
    for (int i = tid; i < p.B; i += SMP_THREADS) {
      const int of = kind(i);
      if ((int)(at >> of & 0xffff) == b) s.row = i;
      at += 1ULL << of;
    }
    __syncthreads();
    b = s.row;
    if (b < 0) return;                            // (more CTAs than rows)
  }
  ctas = group.ctas;
  const int rank = group.rank, per_cta = ctas > 1 ? p.slice : V;
  SmpSlice<L> slice = {static_cast<const L*>(p.logits) + b * p.stride, min(V, rank * per_cta), min(V, (rank + 1) * per_cta), p.vec};
  slice.copied = slice.end - (slice.end - slice.begin) % (16 / (int)sizeof(L));
  const double T = p.temperature ? smp_double(p.temperature[b]) : p.temperature0;
  double top_p = p.top_p ? smp_double(p.top_p[b]) : p.top_p0, min_p = p.min_p ? smp_double(p.min_p[b]) : p.min_p0;
  int top_k = p.top_k ? p.top_k[b] : p.top_k0;
  const bool greedy = !(T > 0.0);
  if (top_k <= 0 || top_k >= V) top_k = 0;
  const bool nucleus = top_p < 1.0;               // (NaN: off)
  top_p = fmax(top_p, 0.0);
  min_p = min_p > 0.0 ? fmin(min_p, 1.0) : 0.0;
  const double u = fmin(fmax(smp_double(p.u[b]), 0.0), 1.0);
  unsigned* const halves = reinterpret_cast<unsigned*>(s.sums);   // low and high words of the sums
  SmpWeight weight(greedy ? 1.0 : T, s.table);

  if (!greedy)
    for (int i = tid; i < SMP_TABLE; i += SMP_THREADS) s.table[i] = smp_table.at[i];
  if (top_k && !greedy)
    for (int i = tid; i < SMP_BINS; i += SMP_THREADS) s.sums[i] = 0;

  // ---- the largest logit and its first index
  unsigned top_key = 0;
  int at = V;
  auto largest = [&](int i, const float* l) {
    const unsigned key = smp_key(smp_max4(l));
    if (key > top_key) top_key = key, at = i;
    return key;
  };
  auto stage = [&](int i, const float* l, unsigned least, unsigned past) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned key = smp_key(l[e]);
      if (key - least < past - least) {
        const unsigned x = atomicAdd(&s.staged, 1u);
        if (x < SMP_CAP) s.weight[x] = (u64)key << 32 | (0xffffffffu - (unsigned)(i + e));
      }
    }
  };
  // Where few are kept of a slice that would have to be read from memory again, candidates for the list are staged at once: as many
  // threads as top_k have seen a logit from `bound` on so far.  (50 largest, with a pass of its own for the list / without: 256 rows of
  // 102400 48 / 41 us, 512 of 128256 109 / 88.  With more than a fourth of the threads that bound is low, and so is min_p of the largest
  // logit so far: 60 / 62 for 256 rows with that alone.)
  const bool streams = !greedy && top_k > 0 && top_k <= SMP_FEW && slice.streams();
  unsigned bound = SMP_LOWEST + 1;
  if (!streams) {
    slice.pass(s, p.status, largest);
  } else {
    if (tid == 0) s.staged = 0;
    __syncthreads();
    slice.pass(
        s, p.status,
        [&](int i, const float* l) {
          if (largest(i, l) >= bound && i >= slice.begin + SMP_CHUNK) stage(i, l, bound, 0xffffffffu);
        },
        [&](int chunk, auto&& sweep) {
          if (chunk & (chunk + 1)) return;        // 0, 1, 3, 7, ...
          unsigned seen = 0;                      // the key that enough threads have seen, but for its last 14 bits
          for (int bit = 31; bit >= 14; --bit)
            if (__syncthreads_count(top_key >= (seen | 1u << bit)) >= top_k) seen |= 1u << bit;
          bound = max(bound, seen);
          if (chunk == 0)
            sweep([&](int i, const float* l) {
              if (smp_key(smp_max4(l)) >= bound) stage(i, l, bound, 0xffffffffu);
            });
        });
  }
  if (greedy && at < V) {                         // which of the four
    float l[4];
    smp_load<L>(slice.row, at, slice.end, 0, l);
    at += smp_key(l[0]) == top_key ? 0 : smp_key(l[1]) == top_key ? 1 : smp_key(l[2]) == top_key ? 2 : 3;
  }
  if (top_k && !greedy) {
    __syncthreads();
    if (top_key) atomicAdd(halves + 2 * (top_key >> 21), 1u);
  }
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
    group.peer(s.tops, tid)[rank] = best;
    group.peer(s.bounds, tid)[rank] = streams && s.staged <= SMP_CAP ? bound : 0;
  }
  group.sync();
  u64 best = 0;
  for (int c = 0; c < ctas; ++c) best = max(best, s.tops[c]);
  unsigned staged_from = 0;                       // all candidates from this key on are staged: 0, they are not
  if (streams) {
    bool all = true;
    for (int c = 0; c < ctas; ++c) {
      all &= s.bounds[c] > 0;
      staged_from = max(staged_from, s.bounds[c]);
    }
    if (!all) staged_from = 0;
  }
  const float top = smp_logit((unsigned)(best >> 32));
  at = V - (int)(unsigned)best;
  if (greedy || top == -INFINITY || s.dead) {
    if (rank == 0 && tid == 0) p.out[b] = top == -INFINITY || s.dead ? -1 : at;
    if (greedy || top == -INFINITY) return;       // (the cluster agrees on these)
  }
  weight.begin(top);
  auto place = [&](u64 total) {                   // the sum that the drawn token's passes
    const u64 x = (u64)(u * (double)total);
    return x < total ? x : total - (total > 0);
  };
  // Logits whose keys are from `least` on and below `past` go to the first CTA's list, by way of one in each CTA; the number of them, in
  // every CTA.
  auto gather = [&](unsigned least, unsigned past, bool staged) {
    constexpr int EACH = SMP_CAP / SMP_THREADS;
    u64 mine[EACH];
    unsigned place[EACH];
    if (tid == 0) s.listed = 0;
    if (!staged) {
      if (tid == 0) s.staged = 0;
      __syncthreads();
      slice.pass(s, p.status, [&](int i, const float* l) {
        if (smp_key(smp_max4(l)) >= least) stage(i, l, least, past);
      });
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < EACH; ++x) {
      place[x] = x * SMP_THREADS + tid;
      mine[x] = place[x] < s.staged ? s.weight[place[x]] : 0;
    }
    if (staged) {                                 // from a lower bound
#pragma unroll
      for (int x = 0; x < EACH; ++x) {
        if (mine[x] >> 32 < least) mine[x] = 0;
        if (mine[x]) place[x] = atomicAdd(&s.listed, 1u);
      }
      __syncthreads();
    }
    if (tid < ctas) group.peer(s.tot, tid)[rank] = staged ? s.listed : s.staged;
    group.sync();
    u64 n = 0, base = 0;
    for (int c = 0; c < ctas; ++c) {
      if (c == rank) base = n;
      n += s.tot[c];
    }
    u64* const list = group.peer(s.list, 0);
    if (n <= SMP_CAP) {
#pragma unroll
      for (int x = 0; x < EACH; ++x)
        if (mine[x]) list[base + place[x]] = mine[x];
    }
    group.sync();
    return n;
  };

  unsigned least_key = 0;                         // smallest key that min_p leaves
  if (min_p > 0.0) {
    const float guess = __double2float_rd(smp_double(top) + log(min_p) * T);
    const unsigned at_guess = min(max(smp_key(guess), SMP_LOWEST + 20), (unsigned)(best >> 32));
    auto passes = [&](unsigned key) { return weight.real(smp_logit(key)) >= min_p; };
    unsigned low = at_guess - 16, high = min(at_guess + 16, (unsigned)(best >> 32));
    if (!passes(high)) high = (unsigned)(best >> 32);
    if (passes(low)) low = SMP_LOWEST - 1;
    least_key = smp_first_key(low, high, passes);
  }
  unsigned border = 0;                            // smallest key kept, and how many of it (those above it all)
  u64 of_border = 0;
  if (top_k || min_p > 0.0) {
    unsigned from = least_key;
    bool few = true;
    if (staged_from) {
      from = max(from, staged_from);
    } else if (top_k) {
      smp_find(s, group, [&](u64 all) { return min((u64)top_k, all + 1); });
      if (s.found[2] >= (u64)top_k) from = max(from, (unsigned)s.found[0] << 21);
      else few = min_p > 0.0 || V <= SMP_CAP;
    }
    const u64 n_list = few ? gather(from, 0xffffffffu, staged_from > 0) : SMP_CAP + 1;
    if (n_list <= SMP_CAP) {
      if (rank > 0) return;
      // ---- one CTA sorts them and finishes
      const int n = (int)n_list;
      smp_sort(s.list, n);
      int kept = max(top_k ? min(n, top_k) : n, 1);
      for (int i = tid; i < kept; i += SMP_THREADS) s.weight[i] = weight(smp_logit((unsigned)(s.list[i] >> 32)));
      __syncthreads();
      smp_scan(s, kept);
      if (nucleus) {
        const u64 want = __double2ull_ru(top_p * (double)s.weight[kept - 1]);
        u64 in = 0;
        for (int i = tid; i < kept; i += SMP_THREADS) in += i == 0 || s.weight[i - 1] < want;
        kept = max((int)smp_block_sum(in, s.warp), 1);
      }
      const u64 target = place(s.weight[kept - 1]);
      __syncthreads();
      for (int i = tid; i < kept; i += SMP_THREADS) {
        const u64 x = s.list[i];
        s.list[i] = x << 32 | x >> 32;            // by index now
      }
      smp_sort(s.list, kept);
      for (int i = tid; i < kept; i += SMP_THREADS) s.weight[i] = weight(smp_logit((unsigned)s.list[i]));
      __syncthreads();
      smp_scan(s, kept);
      for (int i = tid; i < kept; i += SMP_THREADS)
        if (s.weight[i] > target && (i == 0 || s.weight[i - 1] <= target)) p.out[b] = 0xffffffffu - (unsigned)(s.list[i] >> 32);
      return;
    }
  }

  auto clear = [&]() {
    __syncthreads();
    for (int i = tid; i < SMP_BINS; i += SMP_THREADS) s.sums[i] = 0;
    __syncthreads();
  };
  auto add_weight = [&](int bin, u64 w) {         // the carry from the low to the high word is this thread's to see
    const unsigned high = (unsigned)((w + atomicAdd(halves + 2 * bin, (unsigned)w)) >> 32);
    if (high) atomicAdd(halves + 2 * bin + 1, high);
  };
  // The key at which the sum (of the weights above the border so far, or of ones) reaches `target`, and what lies above it.
  auto bit_by_bit = [&](bool weights, u64 target, u64& above) {
    unsigned key_so_far = 0;
    above = 0;
    for (int shift = 21;; shift = shift == 21 ? 10 : 0) {
      const int bits = shift == 0 ? 10 : 11;
      clear();
      slice.pass(s, p.status, [&](int i, const float* l) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned key = smp_key(l[e]);
          if (shift < 21 && key >> (shift + bits) != key_so_far >> (shift + bits)) continue;
          const unsigned bin = key >> shift & ((1u << bits) - 1);
          if (!weights) atomicAdd(halves + 2 * bin, 1u);
          else if (key > border) add_weight(bin, weight(l[e]));
        }
      });
      smp_find(s, group, [&](u64 all) { return min(target - above, all); });
      key_so_far |= (unsigned)s.found[0] << shift;
      above += s.found[1];
      if (shift == 0) return key_so_far;
    }
  };
  if (top_k) {
    u64 above;
    border = bit_by_bit(false, top_k, above);
    of_border = top_k - above;
  }
  if (least_key > border) {                       // (the border's own do not pass min_p)
    border = least_key - 1;
    of_border = 0;
  }
  if (nucleus) {
    const u64 each = of_border ? weight(smp_logit(border)) : 0;
    const float border_logit = border ? smp_logit(border) : -INFINITY;
    clear();
    weight.either([&](auto slow) {
      slice.pass(s, p.status, [&](int i, const float* l) {
        u64 w[4];
        int bin[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = weight.of<decltype(slow)::value>(l[e], bin[e], smp_above(l[e], border_logit));
          bin[e] = weight.bin(bin[e]);
        }
        unsigned old[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) old[e] = w[e] ? atomicAdd(halves + 2 * bin[e], (unsigned)w[e]) : 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned high = (unsigned)((w[e] + old[e]) >> 32);
          if (high) atomicAdd(halves + 2 * bin[e] + 1, high);
        }
      });
    });
    u64 want = 0;
    smp_find(s, group, [&](u64 all) {
      want = max(__double2ull_ru(top_p * (double)(all + each * of_border)), 1ULL);
      if (!each) want = min(want, all);
      return want;
    });
    if (want > s.found[2]) {                      // among those of the border
      of_border = min(of_border, (want - s.found[2] + each - 1) / max(each, 1ULL));
    } else {
      const int bin = (int)s.found[0];
      const u64 above = s.found[1];
      if (warp < 2) {                             // the bin's smallest key, and the next one's
        const int of = bin + warp;
        const unsigned key = of >= SMP_BINS ? 0xffffffffu : smp_first_key(SMP_LOWEST, SMP_HIGHEST, [&](unsigned k) {
          return weight.bin(weight.step(smp_logit(k))) >= of;
        });
        if (lane == 0) s.range[warp] = key;
      }
      __syncthreads();
      const u64 n_list = gather(max(s.range[0], border + 1), s.range[1], false);
      if (n_list <= SMP_CAP) {
        if (rank == 0) {
          const int n = (int)n_list;
          smp_sort(s.list, n);
          for (int i = tid; i < n; i += SMP_THREADS) s.weight[i] = weight(smp_logit((unsigned)(s.list[i] >> 32)));
          __syncthreads();
          smp_scan(s, n);
          for (int i = tid; i < n; i += SMP_THREADS)
            if (above + s.weight[i] >= want && (i == 0 || above + s.weight[i - 1] < want)) {
              const unsigned key = (unsigned)(s.list[i] >> 32);
              int of = 1;
              while (of <= i && (unsigned)(s.list[i - of] >> 32) == key) ++of;
              for (int c = 0; c < ctas; ++c) *group.peer(&s.border, c) = key, *group.peer(&s.of_border, c) = of;
            }
        }
        group.sync();
        border = s.border;
        of_border = s.of_border;
      } else {
        u64 over;
        const unsigned key = bit_by_bit(true, want, over);
        const u64 w = max(weight(smp_logit(key)), 1ULL);
        of_border = (want - over + w - 1) / w;
        border = key;
      }
    }
  }

  // ---- the token: sums of the slices, of the warps' parts of the one it lies in, then along that part
  const u64 each = of_border ? weight(smp_logit(border)) : 0;
  const int part = ((slice.end - slice.begin + SMP_WARPS - 1) / SMP_WARPS + 127) / 128 * 128;
  const int from = min(slice.end, slice.begin + warp * part), to = min(slice.end, from + part);
  auto load = [&](int i, float* l) {              // four logits of a lane
    if (slice.kept && i + 4 <= min(to, slice.copied)) smp_load<L>(reinterpret_cast<const L*>(s.ring), i - slice.begin, to - slice.begin, 1, l);
    else if (i < to) smp_load<L>(slice.row, i, to, slice.vec && (from & 3) == 0, l);
  };
  const float border_logit = border ? smp_logit(border) : -INFINITY;
  auto add = [&](auto slow, const float* l, u64& sum, unsigned& equal) {      // (-inf, behind the end, weighs nothing)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      int j;
      sum += weight.of<decltype(slow)::value>(l[e], j, smp_above(l[e], border_logit));
    }
    if (of_border)
#pragma unroll
      for (int e = 0; e < 4; ++e) equal += smp_same(l[e], border_logit);
  };
  // A warp's part goes by blocks of 512, whose sums are kept (two for a lane, V / 16 / 512 of them at most).
  constexpr int BLOCK = 512, MOST = (1 << 18) / SMP_WARPS / BLOCK + 1;
  static_assert(MOST <= 64 && MOST * SMP_WARPS <= SMP_CAP, "");
  u64 *const sums = s.weight + warp * MOST, *const ties = s.list + warp * MOST;
  u64 sum = 0;
  u64 equal = 0;
  __syncthreads();                                // (the first CTA's lists have been read)
  weight.either([&](auto slow) {
    for (int i = from + lane * 4, k = 0; i - lane * 4 < to; i += BLOCK, ++k) {
      float l[4][4];
      u64 mine = 0;
      unsigned same = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        l[x][0] = l[x][1] = l[x][2] = l[x][3] = -INFINITY;
        load(i + x * 128, l[x]);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) add(slow, l[x], mine, same);
      mine = smp_warp_sum(mine);
      if (of_border) same = __reduce_add_sync(0xffffffffu, same);
      sum += mine;
      equal += same;
      if (lane == 0) sums[k] = mine, ties[k] = same;
    }
  });
  __syncthreads();
  if (lane == 0) s.warp[warp] = sum, s.warp2[warp] = equal;
  __syncthreads();
  if (tid < ctas) {
    u64 x = 0, y = 0;
    for (int w = 0; w < SMP_WARPS; ++w) x += s.warp[w], y += s.warp2[w];
    group.peer(s.tot, tid)[rank] = x;
    group.peer(s.ties, tid)[rank] = y;
  }
  group.sync();
  auto upto = [&](u64 x, u64 y) { return x + each * min(y, of_border); };
  u64 x = 0, y = 0;
  for (int c = 0; c < ctas; ++c) x += s.tot[c], y += s.ties[c];
  const u64 target = place(upto(x, y));
  x = y = 0;
  for (int c = 0; c < rank; ++c) x += s.tot[c], y += s.ties[c];
  for (int w = 0; w < warp; ++w) x += s.warp[w], y += s.warp2[w];
  if (upto(x, y) > target || upto(x + sum, y + equal) <= target) return;
  int i0 = from;
  for (int k = 0; i0 + BLOCK < to && upto(x + sums[k], y + ties[k]) <= target; ++k, i0 += BLOCK) x += sums[k], y += ties[k];
  for (; i0 < to; i0 += 128) {
    const int i = i0 + lane * 4;
    float l[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    load(i, l);
    u64 mine = 0;
    unsigned same = 0;
    weight.either([&](auto slow) { add(slow, l, mine, same); });
    const u64 all = smp_warp_sum(mine);
    const unsigned all_same = __reduce_add_sync(0xffffffffu, same);
    if (upto(x + all, y + all_same) > target) {
      u64 before = mine, before_same = same;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 a = __shfl_up_sync(0xffffffffu, before, o), c = __shfl_up_sync(0xffffffffu, before_same, o);
        if (lane >= o) before += a, before_same += c;
      }
      const unsigned past = __ballot_sync(0xffffffffu, upto(x + before, y + before_same) > target);
      if (lane == __ffs(past) - 1) {
        x += before - mine;
        y += before_same - same;
        for (int e = 0; e < 4 && i + e < to; ++e) {
          const unsigned key = smp_key(l[e]);
          if (border && key <= border) y += key == border;
          else x += weight(l[e]);
          if (upto(x, y) > target) {
            p.out[b] = i + e;
            break;
          }
        }
      }
      return;
    }
    x += all;
    y += all_same;
  }
}

// How many clusters of that many CTAs the current device holds at once.
template <typename L>
static cudaError_t sample_clusters(int device, int ctas, int* most) {
  static std::atomic<int> known[32][5];               // by device and ctas / 4 (0, 1, 2, 4); 0: not asked yet
  std::atomic<int>* const at = device < 32 ? &known[device][ctas / 4] : nullptr;
  if (at && (*most = at->load(std::memory_order_relaxed)) > 0) return cudaSuccess;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(SMP_THREADS);
  cfg.dynamicSmemBytes = sizeof(SmpShared);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaOccupancyMaxActiveClusters(most, sample_kernel<L>, &cfg);
  if (at && e == cudaSuccess) at->store(*most, std::memory_order_relaxed);
  return e;
}

template <typename L>
static int launch_sample(SampleParams p, cudaStream_t stream) {
  auto* f = sample_kernel<L>;
  static std::atomic<unsigned> ready{0};              // a bit for each device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device > 31 || !(ready.load(std::memory_order_relaxed) >> device & 1))) {
    e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SmpShared));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && device <= 31) ready.fetch_or(1u << device, std::memory_order_relaxed);
  }
  // CTAs to a row: as many as leave all rows under way at once, with 2048 logits or more to a CTA.  A GPC's SMs bound what clusters fit:
  // 16 rows of 16 CTAs or 37 of 8 do not, though the SMs hold 296 CTAs.  us after a flushed L2, by this rule / with twice the CTAs, rows
  // of 128256: 16 rows, 50 largest 35 / 41, nucleus 70 / 92; 37 rows, 35 / 47, 90 / 116; 64 rows, 37 / 61, 94 / 127.
  // Rows with settings of their own take unequal times, a nucleus of a flat distribution ten times a greedy row's.  Two waves of
  // clusters even that out (64 rows of 128256, a third without a small k, some of them without a filter, 76 us, one wave 92; 256 rows 131
  // and 191).
  // Where a batch fills the SMs with clusters of four, or with a CTA to a row, long rows take clusters of four and the others a CTA
  // each.  us after a flushed L2, such a mix, 50 largest, a nucleus for every row; that way and by waves, of 128256 logits:
  //   64 rows 88 / 76, 43 / 64, 94 / 119;  192 rows 92 / 128, 53 / 70, 305 / 239;  256 rows 99 / 131, 55 / 79, 317 / 266;
  // of 32000: 64 rows 57 / 54, 29 / 51, 53 / 80;  192 rows 57 / 70, 35 / 48, 120 / 102;  256 rows 57 / 70, 35 / 53, 123 / 116;
  // and not (measured in an earlier form) 96 rows of 128256 72 / 72, 42 / 53, 218 / 132;  512 rows 198 / 193, 92 / 91, 522 / 444.
  // It loses where every row is long, by 28 % at 192 rows of a nucleus each: how many are is on the device.
  auto fit = [&](int n) {
    int most = 0;
    if (e == cudaSuccess) e = sample_clusters<L>(device, n, &most);
    return (long long)most;
  };
  p.unequal = (p.temperature || p.top_k || p.min_p) && p.B <= 1024;      // (each CTA looks at every row's settings)
  int ctas = 1;
  long long clusters = p.B;
  if (p.unequal && p.V >= 4 * 2048 && p.B > fit(8) && p.B <= 3 * fit(2) && (p.B <= fit(4) || p.B > fit(2))) {
    ctas = 4;
    p.whole = (int)min(max(fit(4), 1LL), (long long)p.B);
    clusters = p.whole + (p.B - p.whole + ctas - 1) / ctas;
  } else {
    while (ctas < 16 && p.V / (ctas * 2) >= 2048 && p.B <= (p.unequal ? 2 : 1) * fit(ctas * 2)) ctas *= 2;
  }
  p.slice = ((p.V + ctas - 1) / ctas + 7) / 8 * 8;
  if (e == cudaSuccess) e = chain_clusters(f, ctas, dim3((unsigned)(clusters * ctas)), SMP_THREADS, sizeof(SmpShared), stream, p, ctas);
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
  const int elt = bf16 ? 2 : 4;
  SampleParams p = {logits, stride, u, temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0, B, V,
                    0, 0, 0, out, 0, status_block()};
  p.vec = (reinterpret_cast<uintptr_t>(logits) % (4 * elt) == 0 && stride % 4 == 0) +
          (reinterpret_cast<uintptr_t>(logits) % 16 == 0 && stride * elt % 16 == 0);
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return bf16 ? launch_sample<__nv_bfloat16>(p, stream) : launch_sample<float>(p, stream);
}
