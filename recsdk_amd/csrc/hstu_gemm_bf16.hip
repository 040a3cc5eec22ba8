// The products of hstu_gemm.h for __bf16 operands.
#include "hstu_gemm.h"

namespace hstu {
hipError_t launch_gemm_bf16(const GemmArgs& a, int kind, int tile, hipStream_t st) { return launch_gemm_t<__bf16>(a, kind, tile, st); }
}  // namespace hstu
