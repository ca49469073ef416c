// linear.cu — products of the serving group: which kernel a call takes.
#include "linear.cuh"

namespace mb {

namespace {
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}
bool on(const void* p, long long row_bytes, int bytes) { return reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes) == 0 && row_bytes % bytes == 0; }
}  // namespace

int make_operand_map(CUtensorMap* map, const void* base, int type, long long rows, int n_in, long long stride, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(MIMIR_B200_E_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const int size = type_bytes(type);
  // (the distance of a single row to the next is the caller's to leave open)
  const long long apart = rows > 1 ? stride * size : (static_cast<long long>(n_in) * size + 15) / 16 * 16;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(n_in), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(apart)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(LIN_BLOCK / size), static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
  const CUresult r = fn(map, size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MIMIR_B200_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return MIMIR_B200_OK;
}

int make_result_map(CUtensorMap* map, const void* base, int type, long long rows, int n_out, long long stride) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(MIMIR_B200_E_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const int size = type_bytes(type);
  const long long apart = rows > 1 ? stride * size : (static_cast<long long>(n_out) * size + 15) / 16 * 16;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(n_out), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(apart)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(64 / size), 32}, steps[2] = {1, 1};
  const CUresult r = fn(map, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box, steps,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(MIMIR_B200_E_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return MIMIR_B200_OK;
}

int launch_linear(const MimirLinear& a, bool gated, cudaStream_t st) {
  LinearParams p = {};
  const int size = type_bytes(a.out_type);
  p.x_scale = a.x_scale, p.w_scale = a.w_scale, p.up_scale = a.up_scale, p.bias = a.bias, p.up_bias = a.up_bias;
  p.residual = static_cast<const char*>(a.residual), p.out = static_cast<char*>(a.out);
  p.residual_row = a.residual_stride * size, p.out_row = a.out_stride * size;
  p.rows = a.rows, p.n_out = a.n_out, p.out_type = a.out_type, p.act = a.activation;
  p.kblocks = linear_kblocks(a);
  p.chunk = linear_chunk(a);
  p.formats = a.type == MIMIR_B200_T_BF16 ? (1u << 7) | (1u << 10) : 0u;  // (half, E4M3: 0)
  p.vec_out = on(a.out, p.out_row, 16), p.vec_res = on(a.residual, p.residual_row, 16);
  p.err_word = ctx().dev_error_word;
  return linear_rows_us(a, gated) <= linear_tiles_us(a, gated) ? launch_linear_rows(a, p, gated, st) : launch_linear_tiles(a, p, gated, st);
}

}  // namespace mb
