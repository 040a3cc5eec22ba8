// The products of hstu_gemm.h for _Float16 operands.
#include "hstu_gemm.h"

namespace hstu {
hipError_t launch_gemm_f16(const GemmArgs& a, int kind, int tile, hipStream_t st) { return launch_gemm_t<_Float16>(a, kind, tile, st); }
}  // namespace hstu
