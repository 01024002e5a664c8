// Attention of one new token per sequence over a paged cache of keys and values, grouped heads.
//
//   o[b, h] = sum_i softmax_i(scale * q[b, h] . K[i, h / G]) V[i, h / G],   i over the visible tokens of sequence b:
//   all `lengths[b]` of them, or the last `window`; scores may be capped (cap * tanh(s / cap)).
//
// Every cached row is read once per 16 query heads that share it: 2 * 16 operations a byte at most, so memory bounds it, and
// what the kernel is built for is to keep loads under way on every SM from the first to the last token.
//
// * The work is cut into steps: 32 or 64 tokens of one sequence, for one key head and up to 16 of its query heads.  In the order
//   sequence, head, token they form one list, of which every CTA (one per SM) takes an equal, contiguous part, and every warp of
//   it an equal part of that; how long the sequences are only the device knows, so each CTA adds up the lengths itself.  Where a
//   (sequence, head) goes on in the next warps, the warp that began it waits for them at the kernel's end and joins their
//   running maxima, sums and unnormalised results with its own; where it goes on in the next CTAs, paged_join_kernel does.  A CTA
//   has at most two of the latter, so the scratch is bounded by the grid and not by the batch.  Nothing is added by atomics: the
//   order of every sum follows from the lengths.  (Eight warps sharing units of 256 tokens met in a block barrier wherever a
//   sequence ended: 24 sequences of up to 3001 tokens, 16 heads of 192 / 128 in e4m3, 69 us, the SMs idle for half of it.)
// * A warp has a ring of stages of its own, filled by TMA boxes of 16 tokens (a page is a multiple of 16) that a lane each asks
//   for as soon as it has used a stage up, across the borders of sequences.
// * Scores and weighted sums are mma.sync m16n8k16: the query heads of a key head are its 16 rows.  (A tcgen05 tile would be
//   seven eighths empty, and its operands would still come through shared memory once.)  Statistics and sums are fp32; the
//   weights of the sum are rounded to the operand type of the product, by up to 2^-8 (bf16) or 2^-11 (f16) of each, to
//   either side, against a result that is rounded to bf16 itself; the sum of the weights is not rounded.  f16 ends sooner: weights
//   below 2^-29 of the largest are rounded by up to 2^-40 of that.  (What counts is weight times power of two of the values.  A row
//   of zeros is held with the power 1, others of ordinary size with 2^-7 or so: beside a token of zeros that has nearly all the
//   weight, others of 2^-26 of it are off by up to 2^-7 of themselves.)
// * An e4m3 cache is turned into f16 in registers, exactly; queries become f16 with a power of two for each head that puts the
//   largest at 2^14 (f16 has more bits than bf16; what falls below 2^-38 of the largest is lost).  The keys' powers of two
//   multiply the scores, the values' are added to the exponent of the weights, so that no weight overflows: o = sum_i 2^(s_i + e_i
//   - m) v_i / sum_i 2^(s_i - m) with m the maximum of s_i + max(e_i, -100), so that a token adds 2^100 at most to the
//   lower sum.  K's columns go to the product in another order than Q's would (four neighbouring bytes to a lane instead of two and two);
//   the queries are loaded in the same one.

#include <atomic>

#include "common.cuh"
#include "tpb.h"

namespace tpb {

int sm_count();
int make_tmap_pages(CUtensorMap* map, const void* ptr, int elem_bytes, uint64_t d, uint64_t page, uint64_t heads, uint64_t pages,
                    uint64_t row_stride, uint64_t head_stride, uint64_t page_stride);

struct PagedDecode {
  const __nv_bfloat16* q;
  long long q_b, q_h;                      // strides
  __nv_bfloat16* out;                      // [B, Hkv * G, DV]
  const int* table;
  long long table_b;
  const int* lengths;
  const uint8_t *k_scale, *v_scale;        // a row's scales are contiguous within a page
  long long ks_page, ks_head, vs_page, vs_head;
  float* part_o;                           // [2 to a CTA, then one to a warp][rows][DV]
  float* part_ml;                          // the same [rows][2]: running maximum in log2 units, sum
  int4* split;                             // [CTAs] of the (sequence, head block) that begins in a CTA and goes on: last CTA, slot; or -1
  int* status;
  int B, Hkv, G, blocks, rows;             // blocks of up to 16 query heads to a key head; rows of the largest block
  int pages, page, width, capacity;        // entries of a row of the table, tokens that it can name
  int window, stages, aligned;
  float scale_log2, cap_log2;              // cap_log2: the cap in log2 units, 0 for none
};


struct PagedShape {
  int keys, warps;         // tokens of a warp's step, warps to a CTA
};
// One CTA takes the SM's shared memory, a warp at least one stage of it: many warps with one stage each keep as many bytes under way
// as few with several, and hide the conversions of an 8-bit cache better.  us, as the kernel grew, 64 sequences of up to 8192 tokens, 64 / 8
// heads of 128 in e4m3: 4 warps 159, 8 118, 16 (scores transposed) 90; 128 of 32 / 8 heads in bf16: 4 warps 277, 6 266, 8 261.  Narrow
// heads take 64 tokens to a step, 32 / 64: 64 sequences of 8 / 8 heads of 64 columns, up to 8192 tokens, bf16 82 / 76 us, e4m3 65 / 58, up
// to 4096 50 / 44 and 42 / 37.  That costs wide ones their registers or stages, but an 8-bit cache with more than 8 query heads to
// a key head has to: a part of a result would not fit into a stage of 32.  With more than 8 query heads eight warps have registers
// (64 / 2 heads of 192 / 128 in e4m3: 8 warps 35 us, 10 45, 12 40).
constexpr PagedShape pd_shape(bool held8, bool wide, int width) {
  return {width <= 128 || (held8 && wide && width <= 256) ? 64 : 32, held8 && !wide ? 16 : 8};
}

template <int DK, int DV, bool F8, bool WIDE>
struct PagedTile {
  static constexpr int ELT = F8 ? 1 : 2;
  static constexpr int ROW = 64 * ELT;                       // bytes of a 64-column block's row: the swizzle's width
  static constexpr int BLOCK = 16 * ROW;
  static constexpr int K_BOX = 16 * DK * ELT, V_BOX = 16 * DV * ELT;
  static constexpr int KEYS = pd_shape(F8, WIDE, DK + DV).keys, BOXES = KEYS / 16;
  static constexpr int STAGE = BOXES * (K_BOX + V_BOX);
  static constexpr int SCALES = F8 ? 2 * KEYS : 0;           // of the keys, of the values
  static constexpr int WARPS = pd_shape(F8, WIDE, DK + DV).warps;
};

// Powers of two of 1, for the rows of pages that are not there.
__device__ const uint8_t __align__(16) pd_ones[16] = {127, 127, 127, 127, 127, 127, 127, 127, 127, 127, 127, 127, 127, 127, 127, 127};

__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int row, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %3, %5, %6}], [%2];"
      :
      : "r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(head), "r"(page)
      : "memory");
}
__device__ __forceinline__ void bulk_load_16(uint32_t dst, const void* src, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], 16, [%2];"
               :
               : "r"(dst), "l"(src), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void pd_ldsm(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pd_ldsm_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// d += A (16 x 16) B (16 x 8), operands bf16 or f16
template <bool F16>
__device__ __forceinline__ void pd_mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t e4m3_to_f16(uint32_t v) {      // the low two bytes
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return h;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// The 8 x 8 matrix of 16-bit values that a warp holds two to a lane, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// To 2^-19 of itself: below 1/8, where the other form cancels, by its series (the next term is below 2^-29 of it).
__device__ __forceinline__ float pd_tanh(float x) {
  const float x2 = x * x, small = fmaf(fmaf(fmaf(x2, -17.f / 315, 2.f / 15), x2, -1.f / 3) * x2, x, x);
  const float large = 1.f - __fdividef(2.f, ex2_approx(x * 2.8853900817779268f) + 1.f);
  return fabsf(x) < 0.125f ? small : large;
}

// What is visible of a sequence, in tokens and in steps.
struct Visible {
  int len, lo, first, steps;
};
template <int KEYS>
__device__ __forceinline__ Visible pd_visible(const PagedDecode& p, int b) {
  Visible s;
  s.len = min(max(p.lengths[b], 0), p.capacity);
  s.lo = p.window > 0 ? max(0, s.len - p.window) : 0;
  s.first = s.lo / KEYS;
  s.steps = s.len > 0 ? (s.len - 1) / KEYS - s.first + 1 : 0;
  return s;
}

// Steps of each of `n` CTAs or warps.
__device__ __forceinline__ int pd_share(int steps, int n) { return max(1, (steps + n - 1) / n); }

// A place in the list of steps.
template <int KEYS>
struct PagedCursor {
  int b, hb, at;           // sequence, head block, step of the sequence
  Visible s;
  __device__ __forceinline__ int key0() const { return (s.first + at) * KEYS; }
  __device__ __forceinline__ void next_head(const PagedDecode& p) {
    at = 0;
    if (++hb < p.Hkv * p.blocks) return;
    hb = 0;
    do {
      ++b;
      if (b >= p.B) return;
      s = pd_visible<KEYS>(p, b);
    } while (s.steps == 0);
  }
};

template <int DK, int DV, bool F8, bool WIDE>
__global__ void __launch_bounds__(PagedTile<DK, DV, F8, WIDE>::WARPS * 32, 1)
paged_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const PagedDecode p) {
  using T = PagedTile<DK, DV, F8, WIDE>;
  constexpr int NW = T::WARPS, THREADS = NW * 32, KEYS = T::KEYS, MT = T::BOXES;
  extern __shared__ uint8_t pd_smem_raw[];
  uint8_t* pd_smem = pd_smem_raw + ((1024u - (smem_u32(pd_smem_raw) & 1023u)) & 1023u);
  __shared__ int s_scan[NW], s_at[NW][3], s_ends[NW];
  const int warp = warp_index(), lane = threadIdx.x & 31, ST = p.stages;
  const int HB = p.Hkv * p.blocks;
  uint8_t* ring = pd_smem + (size_t)warp * ST * T::STAGE;
  uint8_t* scales = pd_smem + (size_t)NW * ST * T::STAGE + (size_t)warp * ST * T::SCALES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(pd_smem + (size_t)NW * ST * (T::STAGE + T::SCALES)) + warp * ST;
  const uint32_t ring_at = smem_u32(ring), scales_at = smem_u32(scales);
  if (lane == 0)
    for (int i = 0; i < ST; ++i) mbar_init(&bars[i], 1);
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&k_map);
    tma_prefetch_desc(&v_map);
  }
  fence_barrier_init();
  chain_launch();
  // Lengths, table and queries are read one after the other, each a trip to memory unless something has brought them to L2.
  {
    const int q_lines = DK * 2 / 128, t_lines = (p.width + 31) / 32, n_lines = (p.B + 31) / 32, stride = gridDim.x * THREADS;
    const long long lines = n_lines + (long long)p.B * (t_lines + p.Hkv * p.G * q_lines);
    if (lines <= 8 * stride)
      for (int i = blockIdx.x * THREADS + threadIdx.x; i < lines; i += stride) {
        int x = i - n_lines;
        const void* at = p.lengths + 32 * i;
        if (x >= p.B * t_lines) {
          x -= p.B * t_lines;
          const int row = x / q_lines;
          at = p.q + row / (p.Hkv * p.G) * p.q_b + row % (p.Hkv * p.G) * p.q_h + x % q_lines * 64;
        } else if (x >= 0) {
          at = p.table + x / t_lines * p.table_b + x % t_lines * 32;
        }
        asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
      }
  }
  if (!chain_wait()) return;

  // The list's length, and where this CTA's part and its warps' begin.
  int cta_first = 0, cta_share = 1, cta_steps = 0, share = 1;
  int before = 0, n = 0;                   // of this thread's sequence: steps in front of it (per head block), its own
  auto add_up = [&](int base, int running) {
    const int b = base + threadIdx.x;
    n = b < p.B ? pd_visible<KEYS>(p, b).steps : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = sum;
    __syncthreads();
    before = running + sum - n;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) before += s_scan[w];
      running += s_scan[w];
    }
    return running;
  };
  if (p.aligned) {                         // a CTA for each (sequence, head block)
    const int b = blockIdx.x / HB, own = pd_visible<KEYS>(p, b).steps;
    cta_share = cta_steps = own;
    share = pd_share(own, NW);
    if (lane == 0) s_at[warp][0] = b, s_at[warp][1] = blockIdx.x % HB, s_at[warp][2] = warp * share;
  } else {
    int all = 0;
    for (int base = 0; base < p.B; base += THREADS) all = add_up(base, all);
    cta_share = pd_share(all * HB, gridDim.x);
    cta_first = blockIdx.x * cta_share;
    cta_steps = min(cta_share, all * HB - cta_first);
    share = pd_share(cta_steps, NW);
    for (int base = 0, running = 0; base < p.B; base += THREADS) {
      if (p.B > THREADS) running = add_up(base, running);      // (else as it was left)
      if (n > 0)
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const int in = cta_first + w * share - before * HB;
          if (w * share < cta_steps && in >= 0 && in < n * HB) {
            s_at[w][0] = base + threadIdx.x;
            s_at[w][1] = in / n;
            s_at[w][2] = in % n;
          }
        }
    }
  }
  __syncthreads();
  const int steps = min(share, cta_steps - warp * share);      // (none: 0 or less)
  PagedCursor<KEYS> c = {};
  if (steps > 0) {
    c.b = s_at[warp][0];
    c.hb = s_at[warp][1];
    c.at = s_at[warp][2];
    c.s = pd_visible<KEYS>(p, c.b);
  }
  PagedCursor<KEYS> ahead = c;
  int asked = 0, ask_stage = 0, stage = 0, parity = 0;
  bool alive = true;
  // A lane for each box that holds a visible token: the pages in front of a window may have been given back.  The pages of the step
  // that is asked for next are on their way from the table since the one before was.
  int pg = -1, row = 0;
  bool seen = false;
  auto look_up = [&]() {
    const int key = ahead.key0() + 16 * lane;
    seen = lane < MT && key < ahead.s.len && key + 16 > ahead.s.lo;
    const unsigned at = (unsigned)key / (unsigned)p.page;
    row = key - at * p.page;
    if (seen) pg = p.table[ahead.b * p.table_b + at];
  };
  if (steps > 0) look_up();

  // The fence orders the warp's reads of the stage, in front of the __syncwarp before, ahead of the copy that overwrites it.
  auto ask = [&]() {
    uint64_t* bar = &bars[ask_stage];
    const bool inside = seen && pg >= 0 && pg < p.pages;
    if (seen && !inside) report(p.status, kBadArgument, 72);      // a box outside the pool reads as zeros, of the size 1
    const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, seen)) * (T::K_BOX + T::V_BOX + (F8 ? 32 : 0));
    if (lane == 0) mbar_expect_tx(bar, bytes);
    __syncwarp();
    if (seen) {
      const int head = ahead.hb / p.blocks;
      const uint32_t at = ring_at + ask_stage * T::STAGE;
      fence_proxy_async();
      tma_load_page(at + lane * T::K_BOX, &k_map, bar, row, head, inside ? pg : -1);
      tma_load_page(at + MT * T::K_BOX + lane * T::V_BOX, &v_map, bar, row, head, inside ? pg : -1);
      if (F8) {
        const uint32_t sc = scales_at + ask_stage * T::SCALES + lane * 16;
        bulk_load_16(sc, inside ? p.k_scale + pg * p.ks_page + head * p.ks_head + row : pd_ones, bar);
        bulk_load_16(sc + KEYS, inside ? p.v_scale + pg * p.vs_page + head * p.vs_head + row : pd_ones, bar);
      }
    }
    __syncwarp();
    ++asked;
    if (++ask_stage == ST) ask_stage = 0;
    if (asked >= steps) return;
    if (++ahead.at == ahead.s.steps) ahead.next_head(p);
    look_up();
  };
  while (asked < steps && asked < ST) ask();
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < p.B; b += THREADS)
      if (p.lengths[b] < 0 || p.lengths[b] > p.capacity) report(p.status, kBadArgument, 71);
  if (threadIdx.x == 0 && !p.aligned) p.split[blockIdx.x] = make_int4(-1, 0, 0, 0);
  for (int b = blockIdx.x; b < p.B; b += gridDim.x)        // sequences of no visible token
    if (pd_visible<KEYS>(p, b).steps == 0) {
      uint4* dst = reinterpret_cast<uint4*>(p.out + (long long)b * p.Hkv * p.G * DV);
      for (int i = threadIdx.x; i < p.Hkv * p.G * (DV / 8); i += THREADS) dst[i] = make_uint4(0, 0, 0, 0);
    }

  const int g = lane >> 2, t = lane & 3;
  constexpr int NT = WIDE ? 2 : 1;         // blocks of eight query heads
  constexpr int F16_UP = 15;               // f16 weights are 2^15 times as large: of a long sequence's small ones those from 2^-40 on count
  int done = 0, seg = 0, h0 = 0, rows = 0;
  // Of heads 8 nt + 2t and the one after: columns 16 c + (0 .. 15), two of them to a lane (see column()), maxima and sums.
  float o[NT][DV / 16][4], m[NT][2], l[NT][2];
  bool joins = false;          // this warp's last (sequence, head) goes on in the next one, and it is the one to join them
  auto column = [&](int c, int hi) { return 16 * c + (F8 ? 2 * g + hi : g + 8 * hi); };
  auto put_result = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 8 * nt + 2 * t + x;
        if (r >= rows) continue;
        const float inv = 1.f / l[nt][x];
        __nv_bfloat16* dst = p.out + ((long long)c.b * p.Hkv * p.G + h0 + r) * DV;
#pragma unroll
        for (int cb = 0; cb < DV / 16; ++cb) {
          const uint32_t both = pack_bf16(o[nt][cb][x] * inv, o[nt][cb][2 + x] * inv);
          if constexpr (F8) {
            *reinterpret_cast<uint32_t*>(dst + column(cb, 0)) = both;
          } else {
            reinterpret_cast<uint16_t*>(dst)[column(cb, 0)] = (uint16_t)both;
            reinterpret_cast<uint16_t*>(dst)[column(cb, 1)] = (uint16_t)(both >> 16);
          }
        }
      }
  };
  // A part that another warp or the kernel behind this one joins: results, then maximum and sum of each row.
  struct Part {
    float* o;
    float2* ml;
  };
  auto part_at = [&](int slot) { return Part{p.part_o + (long long)slot * p.rows * DV, reinterpret_cast<float2*>(p.part_ml) + slot * p.rows}; };
  auto warp_part = [&](int w) {            // of a warp of this CTA: in its ring, if it has nothing else to do
    float* o = reinterpret_cast<float*>(pd_smem + (size_t)w * ST * T::STAGE);
    return p.aligned ? Part{o, reinterpret_cast<float2*>(o + (WIDE ? 16 : 8) * DV)} : part_at(2 * gridDim.x + blockIdx.x * NW + w);
  };
  static_assert((WIDE ? 16 : 8) * DV * 4 <= T::STAGE - 16 * 8, "a part fits into a stage");
  auto put_part = [&](const Part& part) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = 8 * nt + 2 * t + x;
        if (r >= rows) continue;
        float* dst = part.o + r * DV;
#pragma unroll
        for (int cb = 0; cb < DV / 16; ++cb) {
          if constexpr (F8) {
            *reinterpret_cast<float2*>(dst + column(cb, 0)) = make_float2(o[nt][cb][x], o[nt][cb][2 + x]);
          } else {
            dst[column(cb, 0)] = o[nt][cb][x];
            dst[column(cb, 1)] = o[nt][cb][2 + x];
          }
        }
        if (g == 0) part.ml[r] = make_float2(m[nt][x], l[nt][x]);
      }
  };
  while (done < steps) {
    seg = min(steps - done, c.s.steps - c.at);
    const int kv_head = c.hb / p.blocks, row0 = (c.hb - kv_head * p.blocks) * 16;
    rows = min(16, p.G - row0);
    h0 = kv_head * p.G + row0;
    // ---- the queries as B operands: head g of each block of eight, two (e4m3: four) neighbouring columns to a register pair
    uint32_t qb[DK / 16][NT][2];
    float qs[NT][2];                       // factors of the scores of heads 2t and 2t + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const __nv_bfloat16* q = p.q + c.b * p.q_b + (h0 + 8 * nt + g) * p.q_h;
      const bool has = 8 * nt + g < rows;
      if constexpr (!F8) {
#pragma unroll
        for (int k = 0; k < DK / 16; ++k) {
          qb[k][nt][0] = has ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 2 * t) : 0;
          qb[k][nt][1] = has ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8 + 2 * t) : 0;
        }
        qs[nt][0] = qs[nt][1] = p.scale_log2;
      } else {
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < DK / 16; ++k) {
          const uint2 a = has ? *reinterpret_cast<const uint2*>(q + k * 16 + 4 * t) : make_uint2(0, 0);
          qb[k][nt][0] = a.x;
          qb[k][nt][1] = a.y;
          most = __vmaxu2(most, __vmaxu2(a.x & 0x7fff7fffu, a.y & 0x7fff7fffu));
        }
        most = max(most & 0xffffu, most >> 16);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = min(max((int)(most >> 7) - 127 - 14, -100), 113);       // the largest becomes 2^14 and more
        const float f = __int_as_float((127 - e) << 23), back = p.scale_log2 * __int_as_float((127 + e) << 23);
        qs[nt][0] = __shfl_sync(0xffffffffu, back, 8 * t);
        qs[nt][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (int k = 0; k < DK / 16; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 v = unpack_bf16(qb[k][nt][x]);
            qb[k][nt][x] = pack_f16(v.x * f, v.y * f);
          }
      }
#pragma unroll
      for (int cb = 0; cb < DV / 16; ++cb) o[nt][cb][0] = o[nt][cb][1] = o[nt][cb][2] = o[nt][cb][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    for (int i = 0; i < seg; ++i) {
      const int key0 = c.key0() + i * KEYS;
      // (a wait that gives up ends the asking; what was asked for is still waited for, each time with a limit)
      if (done + i < asked && !mbar_wait_warp(&bars[stage], parity, p.status, kTimeoutTmaFull, 73)) alive = false;
      const uint32_t k_at = ring_at + stage * T::STAGE, v_at = k_at + MT * T::K_BOX;
      const bool edge = key0 < c.s.lo || key0 + KEYS > c.s.len;
      if (alive) {
        if (edge) {
          // Rows behind the end (or in front of the window) hold anything, NaN too: zeros of the size 1 in the values, -inf in the scores.
          uint4* v = reinterpret_cast<uint4*>(ring + stage * T::STAGE + MT * T::K_BOX);
          for (int x = lane; x < MT * T::V_BOX / 16; x += 32) {
            const int key = key0 + x / (T::V_BOX / 16) * 16 + x % (T::BLOCK / 16) / (T::ROW / 16);
            if (key < c.s.lo || key >= c.s.len) v[x] = make_uint4(0, 0, 0, 0);
          }
          if constexpr (F8)
            for (int x = lane; x < KEYS; x += 32)
              if (key0 + x < c.s.lo || key0 + x >= c.s.len) scales[stage * T::SCALES + KEYS + x] = 127;
          __syncwarp();
        }
        float s[MT][NT][4] = {};
        float factor[MT][2], add[MT][2];     // e4m3: powers of two of the keys, exponents of the values and F16_UP (so m, too)
        if constexpr (F8) {
          const uint8_t* sc = scales + stage * T::SCALES;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            from_e8m0x2(sc[mt * 16 + g] | (uint32_t)sc[mt * 16 + 8 + g] << 8, factor[mt][0], factor[mt][1]);
#pragma unroll
            for (int hi = 0; hi < 2; ++hi)       // (as a multiple of 2^104; 255, NaN: infinity, which makes all results NaN)
              add[mt][hi] = fmaf(__uint_as_float(0x7f7fff01u + sc[KEYS + mt * 16 + hi * 8 + g]), 1.f / (1ULL << 52) / (1ULL << 52),
                                 -(float)((1 << 24) - 255 + 127 - F16_UP));
          }
        }
        // ---- scores, transposed: 16 tokens by 8 heads each; s[mt][nt] = (token g: heads 2t, 2t + 1; token g + 8: the same)
        if constexpr (!F8) {
          const uint32_t at = k_at + ((lane & 7) + ((lane >> 3) & 1) * 8) * 128;
#pragma unroll
          for (int k = 0; k < DK / 16; ++k)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t a[4];
              pd_ldsm(at + mt * T::K_BOX + (k >> 2) * T::BLOCK + ((((k & 3) * 2 + (lane >> 4)) ^ (lane & 7)) << 4), a);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) pd_mma<false>(s[mt][nt], a, qb[k][nt][0], qb[k][nt][1]);
            }
        } else {
          const uint32_t at = k_at + (lane & 7) * 64 + (((lane >> 3) ^ ((lane & 7) >> 1)) << 4);
#pragma unroll
          for (int hf = 0; hf < DK / 64; ++hf)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t lo[4], hi[4];       // tokens 0 - 7 and 8 - 15, 16 columns each
              pd_ldsm(at + mt * T::K_BOX + hf * T::BLOCK, lo);
              pd_ldsm(at + mt * T::K_BOX + hf * T::BLOCK + 512, hi);
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const uint32_t a[4] = {e4m3_to_f16(lo[x]), e4m3_to_f16(hi[x]), e4m3_to_f16(lo[x] >> 16), e4m3_to_f16(hi[x] >> 16)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) pd_mma<true>(s[mt][nt], a, qb[4 * hf + x][nt][0], qb[4 * hf + x][nt][1]);
              }
            }
        }
        // ---- running softmax
        uint32_t pb[MT][NT][2];             // the weights as B operands: token pairs by head
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) top[nt][0] = m[nt][0], top[nt][1] = m[nt][1];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi) {
            const int in = mt * 16 + hi * 8 + g;
            const bool dead = edge && (key0 + in < c.s.lo || key0 + in >= c.s.len);
            const float up = F8 ? fmaxf(add[mt][hi], F16_UP - 100.f) : 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                float v = s[mt][nt][2 * hi + x] * (F8 ? mul_exact(qs[nt][x], factor[mt][hi]) : qs[nt][x]);
                if (p.cap_log2 > 0.f) v = p.cap_log2 * pd_tanh(v / p.cap_log2);
                v = dead ? -INFINITY : v;
                s[mt][nt][2 * hi + x] = v;
                top[nt][x] = fmaxf(top[nt][x], F8 ? v + up : v);
              }
          }
        bool grown = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) top[nt][x] = fmaxf(top[nt][x], __shfl_xor_sync(0xffffffffu, top[nt][x], off));
            grown |= top[nt][x] > m[nt][x];
          }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float a[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              a[x] = top[nt][x] > m[nt][x] ? ex2_approx(m[nt][x] - top[nt][x]) : 1.f;
              l[nt][x] *= a[x];
              m[nt][x] = top[nt][x];
            }
#pragma unroll
            for (int cb = 0; cb < DV / 16; ++cb) {
              o[nt][cb][0] *= a[0]; o[nt][cb][1] *= a[1];
              o[nt][cb][2] *= a[0]; o[nt][cb][3] *= a[1];
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float from[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) from[x] = m[nt][x] == -INFINITY ? 0.f : F8 ? m[nt][x] - F16_UP : m[nt][x];      // (all scores so far are NaN or -inf)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
              float w[2];
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const float v = s[mt][nt][2 * hi + x] - from[x];
                w[x] = ex2_approx(F8 ? v + add[mt][hi] : v);
                l[nt][x] += F8 ? ex2_approx(v) : w[x];
              }
              pb[mt][nt][hi] = transpose_8x8(F8 ? pack_f16(w[0], w[1]) : pack_bf16(w[0], w[1]));
            }
        }
        // ---- weighted sum, transposed: 16 columns by 8 heads
        if constexpr (!F8) {
          const uint32_t at = v_at + ((lane & 7) + (lane >> 4) * 8) * 128;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int cb = 0; cb < DV / 16; ++cb) {
              uint32_t a[4];
              pd_ldsm_t(at + mt * T::V_BOX + (cb >> 2) * T::BLOCK + ((((cb & 3) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4), a);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) pd_mma<false>(o[nt][cb], a, pb[mt][nt][0], pb[mt][nt][1]);
            }
        } else {
          const int vr = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int cp = 0; cp < DV / 32; ++cp) {
              uint32_t b[4];               // tokens 0 - 7 and 8 - 15 of 16 columns, then of the next 16
              pd_ldsm_t(v_at + mt * T::V_BOX + (cp >> 1) * T::BLOCK + vr * 64 + ((((cp & 1) * 2 + (lane >> 4)) ^ ((vr >> 1) & 3)) << 4), b);
#pragma unroll
              for (int x = 0; x < 4; ++x) b[x] = __byte_perm(b[x], 0, 0x3120);      // two tokens of an even column, of the odd one behind it
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const uint32_t a[4] = {e4m3_to_f16(b[2 * x]), e4m3_to_f16(b[2 * x] >> 16), e4m3_to_f16(b[2 * x + 1]), e4m3_to_f16(b[2 * x + 1] >> 16)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) pd_mma<true>(o[nt][2 * cp + x], a, pb[mt][nt][0], pb[mt][nt][1]);
              }
            }
        }
      }
      __syncwarp();                        // the stage has been read
      if (alive && asked < steps) ask();
      if (++stage == ST) {
        stage = 0;
        parity ^= 1;
      }
    }

    // ---- the result, or this warp's part of it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], off);
      if constexpr (F8) {
#pragma unroll
        for (int cb = 0; cb < DV / 16; ++cb)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[nt][cb][x] *= 1.f / (1 << F16_UP);
      }
    }
    const bool starts = c.at == 0, ends = c.at + seg == c.s.steps;
    done += seg;
    if (starts && ends) {
      put_result();
    } else if (!starts && warp > 0) {      // for the warp that began it, or began this CTA's part of it
      put_part(warp_part(warp));
      if (lane == 0) s_ends[warp] = ends;
    } else if (ends) {
      put_part(part_at(2 * blockIdx.x));
    } else {
      joins = true;                        // (the list's part of this warp ends here)
      break;
    }
    c.at += seg;
    if (c.at == c.s.steps) c.next_head(p);
  }
  __syncthreads();
  if (joins) {
    bool ends = false;
    for (int w = warp + 1; w < NW && w * share < cta_steps && !ends; ++w) {
      const Part part = warp_part(w);
      ends = s_ends[w];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int r = 8 * nt + 2 * t + x;
          if (r >= rows) continue;
          const float2 ml = part.ml[r];
          const float* src = part.o + r * DV;
          const float top = fmaxf(m[nt][x], ml.x);
          const float fa = m[nt][x] == -INFINITY ? 0.f : ex2_approx(m[nt][x] - top), fb = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - top);
          m[nt][x] = top;
          l[nt][x] = l[nt][x] * fa + ml.y * fb;
#pragma unroll
          for (int cb = 0; cb < DV / 16; ++cb) {
            const float2 v = F8 ? *reinterpret_cast<const float2*>(src + column(cb, 0)) : make_float2(src[column(cb, 0)], src[column(cb, 1)]);
            o[nt][cb][x] = o[nt][cb][x] * fa + v.x * fb;
            o[nt][cb][2 + x] = o[nt][cb][2 + x] * fa + v.y * fb;
          }
        }
    }
    if (c.at == 0 && ends) {
      put_result();
    } else {
      const int slot = 2 * blockIdx.x + (warp == 0 && done == seg ? 0 : 1);
      put_part(part_at(slot));
      if (c.at == 0 && lane == 0)
        p.split[blockIdx.x] = make_int4((cta_first + warp * share + done - seg + c.s.steps - 1) / cta_share, slot, c.b, c.hb);
    }
  }
}

// Grid (CTAs of the kernel before, rows): joins the parts of the (sequence, head block) that begins in a CTA and goes on, a row to a
// block.  The first part is in the slot that the CTA has noted, the others, which begin with their CTA, in slot 0 of theirs.  What
// a thread reads of the first parts is asked for before their weights are known.
template <int DV>
__global__ void __launch_bounds__(256)
paged_join_kernel(const PagedDecode p) {
  if (!chain_begin()) return;
  constexpr int COLS = DV / 4, SETS = 256 / COLS, AHEAD = 4;
  __shared__ float4 sums[SETS][COLS];
  const int4 split = p.split[blockIdx.x];
  const int f = blockIdx.x, l = split.x, r = blockIdx.y, lane = threadIdx.x & 31;
  const int kv_head = split.w / p.blocks, row0 = (split.w - kv_head * p.blocks) * 16;
  if (l < 0 || r >= p.G - row0) return;
  const int col = threadIdx.x % COLS, set = threadIdx.x / COLS;
  auto slot = [&](int c) { return (c == f ? split.y : 2 * c) * p.rows + r; };
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  auto part = [&](int c) { return *reinterpret_cast<const float4*>(p.part_o + (long long)slot(c) * DV + 4 * col); };
  float4 v[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) v[i] = part(min(f + set + i * SETS, l));
  float top = -INFINITY;
  for (int c = f + lane; c <= l; c += 32) top = fmaxf(top, ml[slot(c)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  auto weight = [&](float m) { return m == -INFINITY ? 0.f : ex2_approx(m - top); };
  float sum = 0.f;
  for (int c = f + lane; c <= l; c += 32) {
    const float2 x = ml[slot(c)];
    sum += weight(x.x) * x.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& x, int c) {
    const float w = weight(ml[slot(c)].x);
    acc.x += w * x.x; acc.y += w * x.y; acc.z += w * x.z; acc.w += w * x.w;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (f + set + i * SETS <= l) add(v[i], f + set + i * SETS);
#pragma unroll 4
  for (int c = f + set + AHEAD * SETS; c <= l; c += SETS) add(part(c), c);
  sums[set][col] = acc;
  __syncthreads();
  if (set == 0) {
    for (int k = 1; k < SETS; ++k) {
      const float4 x = sums[k][col];
      acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
    }
    const float inv = 1.f / sum;
    *(reinterpret_cast<uint2*>(p.out + ((long long)split.z * p.Hkv * p.G + kv_head * p.G + row0 + r) * DV) + col) =
        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
}

static int pd_grid(long long most_steps) {
  const long long sms = sm_count();
  return (int)(most_steps < 1 ? 1 : most_steps < sms ? most_steps : sms);
}

// Whether a CTA takes a whole (sequence, head block), with nothing to add up before and to join behind: short sequences, or as many of
// them as there are SMs.  us in a graph, list / CTA each: 1 sequence of 32 / 8 heads of 128 in bf16, 64 tokens 6.4 / 3.7, 256 6.7 / 6.2,
// 512 7.0 / 7.7; 16 sequences 512 10.9 / 8.0, 1024 11.9 / 10.6, 2048 15.3 / 15.4; 8 of 16 heads of 192 / 128, 1024 12.0 / 10.8, 2048 15.1 / 16.9.
static bool pd_aligned(long long jobs, long long capacity) {
  return jobs <= sm_count() && capacity <= (2 * jobs >= sm_count() ? 1024 : 256);
}

template <int DK, int DV, bool F8, bool WIDE>
static int launch_paged_decode(PagedDecode p, int grid, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t stream) {
  using T = PagedTile<DK, DV, F8, WIDE>;
  constexpr int MOST = 227 * 1024 - 1024 - 1024;      // (static arrays; alignment)
  static_assert(T::WARPS * (T::STAGE + T::SCALES + 8) <= MOST, "every warp has a stage");
  p.stages = MOST / (T::WARPS * (T::STAGE + T::SCALES + 8));
  if (p.stages > 8) p.stages = 8;
  const int smem = 1024 + T::WARPS * p.stages * (T::STAGE + T::SCALES + 8);
  auto* f = paged_decode_kernel<DK, DV, F8, WIDE>;
  static std::atomic<unsigned> ready{0};              // a bit for each device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device > 31 || !(ready.load(std::memory_order_relaxed) >> device & 1))) {
    e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && device <= 31) ready.fetch_or(1u << device, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return 1000 + (int)e;
  chain(f, grid, T::WARPS * 32, smem, stream, km, vm, p);
  if (grid > 1 && !p.aligned) chain(paged_join_kernel<DV>, dim3(grid, p.rows), 256, 0, stream, p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

}  // namespace tpb

using namespace tpb;

// Bytes of scratch for tpb_paged_decode.
extern "C" int tpb_paged_decode_scratch(int B, int Hkv, int G, int DK, int DV, int held8, int capacity) {
  const PagedShape shape = pd_shape(held8 != 0, G > 8, DK + DV);
  const long long jobs = (long long)B * Hkv * ((G + 15) / 16), steps = jobs * (((long long)capacity + shape.keys - 1) / shape.keys);
  return pd_aligned(jobs, capacity) ? 0 : pd_grid(steps) * ((2 + shape.warps) * (G < 16 ? G : 16) * (DV + 2) * 4 + 16);
}

// q [B, Hkv * G, DK] bf16 (strides q_b, q_h), pools as in tpb_paged_rows (strides of pages, tokens, heads; scales contiguous over
// a page's tokens), table [B, table_width] with rows table_b apart, lengths [B]; out [B, Hkv * G, DV] bf16, contiguous.
// window 0: none; softcap 0: none.  scratch: 16-byte aligned.
extern "C" int tpb_paged_decode(const void* q, long long q_b, long long q_h, const void* k_pool, const void* v_pool,
                                const void* k_scale, const void* v_scale, const long long* strides, const int* table, long long table_b,
                                int table_width, const int* lengths, void* out, void* scratch, int B, int Hkv, int G, int DK, int DV,
                                int pages, int page, int window, float scale, float softcap, void* stream_) {
  const bool held8 = k_scale != nullptr;
  const int elt = held8 ? 1 : 2;
  if (B < 0 || B > (1 << 24) || Hkv < 1 || G < 1 || pages < 1 || page < 16 || page % 16 || window < 0 || table_width < 0 || softcap < 0.f) return -2;
  if ((long long)pages * page > 0x7fffffffLL || (long long)Hkv * G > 65535) return -2;
  if (held8 != (v_scale != nullptr)) return -2;
  for (const void* a : {q, k_pool, v_pool, (const void*)out, (const void*)scratch, k_scale, v_scale})
    if (reinterpret_cast<uintptr_t>(a) % 16) return -2;
  if (q_b % 8 || q_h % 8) return -2;
  for (int i = 0; i < 2; ++i) {
    for (int j = 0; j < 3; ++j)
      if (strides[6 * i + j] * elt % 16 || strides[6 * i + j] < 0) return -2;
    if (held8 && (strides[6 * i + 3] % 16 || strides[6 * i + 4] != 1 || strides[6 * i + 5] % 16)) return -2;
  }
  if (B == 0) return 0;
  long long capacity = (long long)table_width * page;
  if (capacity > (long long)0x7fffff00) return -2;
  const int blocks = (G + 15) / 16;
  const PagedShape shape = pd_shape(held8, G > 8, DK + DV);
  const long long steps = (long long)B * Hkv * blocks * ((capacity + shape.keys - 1) / shape.keys);
  if (steps > 0x3fffffffLL) return -2;
  PagedDecode p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_b = q_b;
  p.q_h = q_h;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.table = table;
  p.table_b = table_b;
  p.lengths = lengths;
  p.k_scale = static_cast<const uint8_t*>(k_scale);
  p.v_scale = static_cast<const uint8_t*>(v_scale);
  p.ks_page = strides[3];
  p.ks_head = strides[5];
  p.vs_page = strides[9];
  p.vs_head = strides[11];
  p.aligned = pd_aligned((long long)B * Hkv * blocks, capacity);
  const int grid = p.aligned ? B * Hkv * blocks : pd_grid(steps);
  p.rows = G < 16 ? G : 16;
  const long long part_rows = (long long)grid * (2 + shape.warps) * p.rows;
  p.split = static_cast<int4*>(scratch);
  p.part_o = reinterpret_cast<float*>(p.split + grid);
  p.part_ml = p.part_o + part_rows * DV;
  p.status = status_block();
  p.B = B;
  p.Hkv = Hkv;
  p.G = G;
  p.blocks = blocks;
  p.pages = pages;
  p.page = page;
  p.width = table_width;
  p.capacity = (int)capacity;
  p.window = window;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.cap_log2 = softcap * 1.4426950408889634f;
  CUtensorMap km, vm;
  if (make_tmap_pages(&km, k_pool, elt, DK, page, Hkv, pages, strides[1] * elt, strides[2] * elt, strides[0] * elt)) return -3;
  if (make_tmap_pages(&vm, v_pool, elt, DV, page, Hkv, pages, strides[7] * elt, strides[8] * elt, strides[6] * elt)) return -4;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const bool wide = G > 8;
#define PD_CASE(dk, dv)                                                                                        \
  if (DK == dk && DV == dv)                                                                                    \
    return held8 ? (wide ? launch_paged_decode<dk, dv, true, true>(p, grid, km, vm, stream)                    \
                         : launch_paged_decode<dk, dv, true, false>(p, grid, km, vm, stream))                  \
                 : (wide ? launch_paged_decode<dk, dv, false, true>(p, grid, km, vm, stream)                   \
                         : launch_paged_decode<dk, dv, false, false>(p, grid, km, vm, stream));
  PD_CASE(128, 128)
  PD_CASE(192, 128)
  PD_CASE(64, 64)
#undef PD_CASE
  return -2;
}
