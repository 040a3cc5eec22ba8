// The products of hstu_gemm.h and hstu_gated_rows.h for __bf16 operands.
#include "hstu_gated_rows.h"

namespace hstu {
hipError_t launch_gemm_bf16(const GemmArgs& a, int kind, int tile, hipStream_t st) { return launch_gemm_t<__bf16>(a, kind, tile, st); }
hipError_t launch_gated_rows_bf16(const RowsArgs& a, hipStream_t st) { return launch_gated_rows_t<__bf16>(a, st); }
}  // namespace hstu
