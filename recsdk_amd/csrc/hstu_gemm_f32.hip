// The products of hstu_gemm.h and hstu_gated_rows.h for float operands.
#include "hstu_gated_rows.h"

namespace hstu {
hipError_t launch_gemm_f32(const GemmArgs& a, int kind, int tile, hipStream_t st) { return launch_gemm_t<float>(a, kind, tile, st); }
hipError_t launch_gated_rows_f32(const RowsArgs& a, hipStream_t st) { return launch_gated_rows_t<float>(a, st); }
}  // namespace hstu
