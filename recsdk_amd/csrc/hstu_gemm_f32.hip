// The products of hstu_gemm.h for float operands.
#include "hstu_gemm.h"

namespace hstu {
hipError_t launch_gemm_f32(const GemmArgs& a, int kind, int tile, hipStream_t st) { return launch_gemm_t<float>(a, kind, tile, st); }
}  // namespace hstu
