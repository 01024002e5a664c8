// Host-side construction of TMA tensor maps (cuTensorMapEncodeTiled resolved through the
// runtime's driver entry point, so the library does not link against libcuda).

#include <mutex>

#include "common.cuh"

namespace tpb {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// cuTensorMapEncodeTiled is a driver call and needs the device's primary context to be current on the
// calling thread.  A thread that has only had its device selected (an autograd worker whose first
// operation is one of this library's GEMMs) has none yet: a runtime call binds it, once per thread.
static void bind_context_once() {
  thread_local bool bound = false;
  if (!bound) {
    cudaFree(nullptr);
    bound = true;
  }
}

// 2-D map: dims {inner, outer}, row pitch in elements, box {box_inner, box_outer}, 128B swizzle.
int make_tmap_2d(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t outer, uint64_t pitch_elems,
                 uint32_t box_inner, uint32_t box_outer, int elem_bytes) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return -1;
  bind_context_once();
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {pitch_elems * elem_bytes};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  CUtensorMapDataType dt = elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  CUresult r = fn(map, dt, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)r;
}

// 3-D bf16 map for [rows, heads, d] views of token-major activations: dim0 = d (contiguous),
// dim1 = rows (pitch stride1_elems), dim2 = heads (pitch stride2_elems); box {box0, box1, 1}.
int make_tmap_3d(CUtensorMap* map, const void* ptr, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t stride1_elems,
                 uint64_t stride2_elems, uint32_t box0, uint32_t box1) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return -1;
  bind_context_once();
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {stride1_elems * 2, stride2_elems * 2};
  cuuint32_t box[3] = {box0, box1, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)r;
}

// Map of an output matrix (bf16 or fp32) of `planes` planes of [rows, cols], for stores of 32 rows x 128 bytes.
int make_tmap_out(CUtensorMap* map, const void* ptr, uint64_t cols, uint64_t rows, uint64_t planes, uint64_t ld_elems,
                  uint64_t plane_elems, int elem_bytes) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return -1;
  bind_context_once();
  cuuint64_t dims[3] = {cols, rows, planes};
  cuuint64_t strides[2] = {ld_elems * elem_bytes, plane_elems * elem_bytes};
  cuuint32_t box[3] = {(cuuint32_t)(128 / elem_bytes), 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUtensorMapDataType dt = elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  CUresult r = fn(map, dt, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)r;
}

// Pools of a paged cache: 16 tokens of one page and head, all `d` columns, in blocks of 64 columns [d / 64][16 tokens][64].
// Swizzle over a block's row: 128 bytes of bf16, 64 of 8-bit values.  Strides in bytes.
int make_tmap_pages(CUtensorMap* map, const void* ptr, int elem_bytes, uint64_t d, uint64_t page, uint64_t heads, uint64_t pages,
                    uint64_t row_stride, uint64_t head_stride, uint64_t page_stride) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return -1;
  bind_context_once();
  cuuint64_t dims[5] = {64, page, d / 64, heads, pages};
  cuuint64_t strides[4] = {row_stride, (cuuint64_t)(64 * elem_bytes), head_stride, page_stride};
  cuuint32_t box[5] = {64, 16, (cuuint32_t)(d / 64), 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  CUresult r = fn(map, elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(ptr), dims,
                  strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, elem_bytes == 2 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)r;
}

}  // namespace tpb
