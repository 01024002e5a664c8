// Keys and values in a paged cache: rows written (quantised on the way) and read back.
//
// A pool holds P pages of `page` tokens for H heads; a row is one token's D values of one head, contiguous, in bf16 or in
// e4m3 with one power of two for the row.  For a row x the exponent is the smallest e (at least -100) with max |x| <= 448 * 2^e,
// over the finite ones, and the values held are x * 2^-e rounded to nearest even (448 * 2^e for an infinity, NaN stays NaN).
// The factor is a power of two so that nothing but that one rounding is lost: e4m3 has its own exponent, a finer factor would
// move the values within their steps and not the steps, and a row that was read back and written again is the same.  Scale
// bytes are e + 127, the form of e8m0.
//
// Both directions are bound by memory: every value is moved once.  A row is held by 4 to 32 lanes, two or three 16-byte vectors
// each, and a warp takes four sets of rows at once so that their loads are all in flight.  (One vector to a lane, with twice the lanes:
// finding places and the largest value cost twice as many instructions for a byte, 30011 tokens of 8 heads of 128 to e4m3 36 us instead
// of 31, 20000 of 16 of 192 / 128 82 instead of 53, at a copy's rate 28 and 47.)

#include "common.cuh"
#include "tpb.h"

namespace tpb {

// One pool and the rows that go there or come from there (strides in elements; scales: null for bf16).
struct PagedRows {
  __nv_bfloat16* x;
  long long x_token, x_head;
  uint8_t* pool;
  long long page_bytes, row_bytes, head_bytes;
  uint8_t* scale;
  long long s_page, s_row, s_head;
  int D;
};

constexpr int PAGED_THREADS = 256;
// Sets of rows per warp under way together.  (2 / 4: 30011 tokens of 8 heads to e4m3 33 / 31 us.)
constexpr int PAGED_ROWS = 4;

// The larger magnitude of each 16-bit half, as bits; FINITE: among finite bf16 values.
template <bool FINITE>
__device__ __forceinline__ uint32_t max_of(uint32_t m, uint32_t v) {
  v &= 0x7fff7fffu;
  return __vmaxu2(m, FINITE ? v & __vcmpltu2(v, 0x7f807f80u) : v);
}
// Of all values of a row, which LANES lanes hold.
template <bool FINITE, int LANES, int V>
__device__ __forceinline__ uint32_t row_max(const uint4* d) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < V; ++j)
    m = max_of<FINITE>(max_of<FINITE>(max_of<FINITE>(max_of<FINITE>(m, d[j].x), d[j].y), d[j].z), d[j].w);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  return max(m & 0xffffu, m >> 16);
}
// Exponent e of a row whose largest finite magnitude has these bf16 bits; 448 = 1.75 * 2^8.
__device__ __forceinline__ int row_exponent(uint32_t amax) {
  if (amax == 0) return 0;
  return max(-100, (int)(amax >> 7) - 127 - 8 + ((amax & 0x7f) > 0x60 ? 1 : 0));
}

// LANES lanes hold a row, V 16-byte vectors of bf16 each.  Grid y: keys, values.
// WRITE: x -> pool, else pool -> x.  HELD8: the pool is e4m3.
template <int LANES, int V, bool WRITE, bool HELD8>
__global__ void __launch_bounds__(PAGED_THREADS, V > 2 ? 3 : 4)
paged_rows_kernel(PagedRows k, PagedRows v, const long long* __restrict__ slots, unsigned rows, unsigned H, unsigned page,
                  long long n_slots, int* st) {
  if (!chain_begin()) return;
  const PagedRows p = blockIdx.y ? v : k;
  const int per_warp = 32 / LANES, lane = threadIdx.x & 31, in_row = lane % LANES;
  const unsigned warp = blockIdx.x * (PAGED_THREADS / 32) + (threadIdx.x >> 5);
  // A lane finds a row's places for the lanes that move it.  (Both in the form with one vector to a lane, 30011 tokens of 8 heads to e4m3:
  // every lane for its own rows, 50 us instead of 41; eight tokens of one head to a warp, which lie together, instead of eight heads of
  // one token, 37 instead of 36.)
  const unsigned r = warp * (per_warp * PAGED_ROWS) + lane, t = r / H, h = r - t * H;      // (rows < 2^31)
  const bool live = lane < per_warp * PAGED_ROWS && r < rows;
  __nv_bfloat16* const my_x = live ? p.x + (long long)t * p.x_token + (long long)h * p.x_head : nullptr;
  const long long my_slot = live ? slots[t] : -1;
  auto of_row = [&](auto* mine, int i) {
    return reinterpret_cast<decltype(mine)>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), i * per_warp + lane / LANES));
  };
  uint4 d[PAGED_ROWS][V];
  __nv_bfloat16* x[PAGED_ROWS];
#pragma unroll
  for (int i = 0; i < PAGED_ROWS; ++i) {
    x[i] = of_row(my_x, i);
    if (WRITE) {                        // (without waiting for the slot)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = in_row + j * LANES;        // 8 values
        d[i][j] = x[i] != nullptr && c * 8 < p.D ? reinterpret_cast<const uint4*>(x[i])[c] : make_uint4(0, 0, 0, 0);
      }
    }
  }
  uint8_t *my_at = nullptr, *my_sc = nullptr;
  if (my_slot >= 0 && my_slot < n_slots) {
    const unsigned s = (unsigned)my_slot, pg = s / page, off = s - pg * page;
    my_at = p.pool + pg * p.page_bytes + off * p.row_bytes + h * p.head_bytes;
    if (HELD8) my_sc = p.scale + pg * p.s_page + off * p.s_row + h * p.s_head;
  } else if (my_slot != -1) {
    report(st, kBadArgument, 70);
  }
  uint8_t* at[PAGED_ROWS];
  uint8_t* sc[PAGED_ROWS];
#pragma unroll
  for (int i = 0; i < PAGED_ROWS; ++i) {
    at[i] = of_row(my_at, i);
    sc[i] = HELD8 ? of_row(my_sc, i) : nullptr;
    if (!WRITE) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = in_row + j * LANES;
        d[i][j] = make_uint4(0, 0, 0, 0);
        if (at[i] == nullptr || c * 8 >= p.D) continue;
        if (!HELD8) {
          d[i][j] = reinterpret_cast<const uint4*>(at[i])[c];
        } else {
          const uint2 u = reinterpret_cast<const uint2*>(at[i])[c];
          d[i][j].x = u.x;
          d[i][j].y = u.y;
          d[i][j].z = *sc[i];
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PAGED_ROWS; ++i) {
    if (WRITE && HELD8) {
      uint32_t m = row_max<false, LANES, V>(d[i]);
      if (__any_sync(0xffffffffu, m >= 0x7f80u)) m = row_max<true, LANES, V>(d[i]);      // (an infinity or NaN)
      if (at[i] == nullptr) continue;
      const int e = row_exponent(m);
      const float f = __int_as_float((127 - e) << 23);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = in_row + j * LANES;
        if (c * 8 >= p.D) continue;
        const float2 a = unpack_bf16(d[i][j].x), b = unpack_bf16(d[i][j].y), g = unpack_bf16(d[i][j].z), h = unpack_bf16(d[i][j].w);
        uint2 q;
        q.x = to_e4m3x2(a.x * f, a.y * f) | to_e4m3x2(b.x * f, b.y * f) << 16;
        q.y = to_e4m3x2(g.x * f, g.y * f) | to_e4m3x2(h.x * f, h.y * f) << 16;
        reinterpret_cast<uint2*>(at[i])[c] = q;
      }
      if (in_row == 0) *sc[i] = (uint8_t)(e + 127);
    } else {
      if (x[i] == nullptr || (WRITE && at[i] == nullptr)) continue;      // (a read of no slot gives zeros)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int c = in_row + j * LANES;
        if (c * 8 >= p.D) continue;
        uint4 o = d[i][j];
        if (!WRITE && HELD8) {
          float f, none;
          from_e8m0x2(d[i][j].z, f, none);
          const float2 a = from_e4m3x2(d[i][j].x), b = from_e4m3x2(d[i][j].x >> 16), g = from_e4m3x2(d[i][j].y), h = from_e4m3x2(d[i][j].y >> 16);
          o.x = pack_bf16(mul_exact(a.x, f), mul_exact(a.y, f));
          o.y = pack_bf16(mul_exact(b.x, f), mul_exact(b.y, f));
          o.z = pack_bf16(mul_exact(g.x, f), mul_exact(g.y, f));
          o.w = pack_bf16(mul_exact(h.x, f), mul_exact(h.y, f));
        }
        reinterpret_cast<uint4*>(WRITE ? (void*)at[i] : (void*)x[i])[c] = o;
      }
    }
  }
}

template <int LANES, int V>
static void launch_paged_rows(const PagedRows& k, const PagedRows& v, const long long* slots, unsigned rows, int H, int page,
                              long long n_slots, bool write, bool held8, cudaStream_t stream) {
  const long long per_block = (long long)(PAGED_THREADS / 32) * (32 / LANES) * PAGED_ROWS;
  const dim3 grid((unsigned)(((long long)rows + per_block - 1) / per_block), 2);
  auto* f = write ? (held8 ? paged_rows_kernel<LANES, V, true, true> : paged_rows_kernel<LANES, V, true, false>)
                  : (held8 ? paged_rows_kernel<LANES, V, false, true> : paged_rows_kernel<LANES, V, false, false>);
  chain(f, grid, PAGED_THREADS, 0, stream, k, v, slots, rows, H, page, n_slots, status_block());
}

}  // namespace tpb

using namespace tpb;

// Rows of keys (index 0) and values (1): x [T, H, D] bf16 with strides x_strides[2 * i] (token) and [2 * i + 1] (head), pools
// with strides[6 * i ..] = page, token in page, head of the pool and of its scales (all in elements; scales null: bf16 pools).
// slots [T]: token in the pool, page * page_size + offset; -1: no row is written, zeros are read.  Any other value outside the
// pool is left out in the same way and reported in the status block.
extern "C" int tpb_paged_rows(int write, void* k, void* v, void* k_pool, void* v_pool, void* k_scale, void* v_scale,
                              const long long* slots, long long T, int H, int Dk, int Dv, int pages, int page,
                              const long long* x_strides, const long long* strides, void* stream_) {
  const bool held8 = k_scale != nullptr;
  const int elt = held8 ? 1 : 2;
  if (T < 0 || H < 1 || pages < 0 || page < 1 || (long long)pages * page > 0x7fffffffLL || held8 != (v_scale != nullptr)) return -2;
  PagedRows r[2];
  void* xs[2] = {k, v};
  void* pools[2] = {k_pool, v_pool};
  void* scales[2] = {k_scale, v_scale};
  const int D[2] = {Dk, Dv};
  for (int i = 0; i < 2; ++i) {
    if (D[i] < 8 || D[i] % 8 || D[i] > 512 || (held8 && D[i] % 16)) return -2;
    if (reinterpret_cast<uintptr_t>(xs[i]) % 16 || reinterpret_cast<uintptr_t>(pools[i]) % 16) return -2;
    if (x_strides[2 * i] % 8 || x_strides[2 * i + 1] % 8) return -2;
    for (int j = 0; j < 3; ++j)
      if (strides[6 * i + j] * elt % 16) return -2;
    r[i] = {static_cast<__nv_bfloat16*>(xs[i]), x_strides[2 * i], x_strides[2 * i + 1], static_cast<uint8_t*>(pools[i]),
            strides[6 * i] * elt, strides[6 * i + 1] * elt, strides[6 * i + 2] * elt, static_cast<uint8_t*>(scales[i]),
            strides[6 * i + 3], strides[6 * i + 4], strides[6 * i + 5], D[i]};
  }
  if (T == 0) return 0;
  if (T > 0x7fffffffLL / H) return -2;
  const int most = Dk > Dv ? Dk : Dv;
  const long long n_slots = (long long)pages * page;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  auto* launch = most <= 64 ? launch_paged_rows<4, 2> : most <= 128 ? launch_paged_rows<8, 2>
                                            : most <= 192 ? launch_paged_rows<8, 3> : most <= 256 ? launch_paged_rows<16, 2> : launch_paged_rows<32, 2>;
  launch(r[0], r[1], slots, (unsigned)(T * H), H, page, n_slots, write != 0, held8, stream);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
